// token_rows.cuh — what the row operators (norms, 8-bit quantiser) share: a row's values in the registers of its team of
// threads, eight consecutive ones a thread and turn (or neighbours by neighbours where rows are not aligned), and the team's
// sums and maxima.
#pragma once

#include "later.cuh"
#include "pairs.cuh"
#include "token.cuh"

namespace fxk {
namespace {

constexpr int kVec = 8;  // consecutive values of a thread: 16 bytes of a 16-bit type

// Eight 16-bit values, widened. The type's branch lies around the eight, not inside.
__device__ __forceinline__ void unpack8(const uint4& v, int type, float (&f)[kVec]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (type == kTokF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = __half22float2(reinterpret_cast<const __half2&>(w[j]));
            f[2 * j] = t.x;
            f[2 * j + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = __uint_as_float(w[j] << 16);
            f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
}

// A thread's eight values of turn u in a row at p, widened. VEC: consecutive from column (u TEAM + me) 8 on, 16-byte
// aligned; else one of every TEAM columns, so that neighbours read neighbours. Columns past the row are 0.
template <int TEAM, bool VEC>
__device__ __forceinline__ int column(int u, int j, int me) {
    return VEC ? (u * TEAM + me) * kVec + j : (u * kVec + j) * TEAM + me;
}
template <int TEAM, bool VEC, bool CONST>
__device__ __forceinline__ void load8(const void* p, int64_t row, int type, int u, int me, int cols, float (&f)[kVec]) {
    if (VEC) {
        const int c = column<TEAM, VEC>(u, 0, me);
        if (c >= cols) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) f[j] = 0.f;
        } else if (type == kTokF32) {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + row + c);
            const float4 a = CONST ? __ldg(q) : q[0], b = CONST ? __ldg(q + 1) : q[1];
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
            const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + row + c);
            unpack8(CONST ? __ldg(q) : q[0], type, f);
        }
    } else if (type == kTokF32) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            const int c = column<TEAM, VEC>(u, j, me);
            f[j] = c < cols ? static_cast<const float*>(p)[row + c] : 0.f;
        }
    } else {
        uint16_t v[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            const int c = column<TEAM, VEC>(u, j, me);
            v[j] = c < cols ? static_cast<const uint16_t*>(p)[row + c] : uint16_t{0};
        }
        if (type == kTokF16) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) f[j] = __half2float(__ushort_as_half(v[j]));
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j) f[j] = __uint_as_float(static_cast<uint32_t>(v[j]) << 16);
        }
    }
}
template <int TEAM, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t row, int type, int u, int me, int cols, const float (&f)[kVec]) {
    if (VEC) {
        const int c = column<TEAM, VEC>(u, 0, me);
        if (c >= cols) return;
        if (type == kTokF32) {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + row + c);
            q[0] = make_float4(f[0], f[1], f[2], f[3]);
            q[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else if (type == kTokE4M3) {
            uint32_t w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * j], f[4 * j + 1]), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * j + 2], f[4 * j + 3]), __NV_SATFINITE, __NV_E4M3);
                w[j] = lo | hi << 16;
            }
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p) + row + c) = make_uint2(w[0], w[1]);
        } else {
            uint32_t w[4];
            if (type == kTokF16) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
                    w[j] = reinterpret_cast<const uint32_t&>(h);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                    w[j] = reinterpret_cast<const uint32_t&>(h);
                }
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
        auto each = [&](auto* q, auto&& make) {
            q += row;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const int c = column<TEAM, VEC>(u, j, me);
                if (c < cols) q[c] = make(f[j]);
            }
        };
        if (type == kTokF32)
            each(static_cast<float*>(p), [](float v) { return v; });
        else if (type == kTokF16)
            each(static_cast<__half*>(p), [](float v) { return __float2half_rn(v); });
        else if (type == kTokBF16)
            each(static_cast<__nv_bfloat16*>(p), [](float v) { return __float2bfloat16_rn(v); });
        else
            each(static_cast<__nv_fp8_storage_t*>(p), [](float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); });
    }
}

// Sum and maximum over the team; every thread gets them. red: a block's shared memory. Teams inside a warp take part
// together, as all lanes of a warp run through the same rows.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* red) {
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TEAM > 32) {
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
        __syncthreads();
        v = threadIdx.x % 32 < TEAM / 32 ? red[threadIdx.x % 32] : 0.f;
#pragma unroll
        for (int o = TEAM > 512 ? 16 : TEAM > 256 ? 8 : TEAM / 64; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        v = __shfl_sync(0xffffffffu, v, 0);
    }
    return v;
}
template <int TEAM>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t* red) {
    if constexpr (TEAM < 32) {
#pragma unroll
        for (int o = TEAM / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    } else {
        v = __reduce_max_sync(0xffffffffu, v);
    }
    if constexpr (TEAM > 32) {
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
        __syncthreads();
        v = __reduce_max_sync(0xffffffffu, red[threadIdx.x % 32 < TEAM / 32 ? threadIdx.x % 32 : 0]);
    }
    return v;
}

// Rows on their way to shared memory, a thread's own 16 bytes a turn (eight 16-bit values), several rows ahead: no registers are
// held for them and no thread waits for another's. slot: a thread's 16 bytes of one row and tensor.
__device__ __forceinline__ void copy16(uint4* slot, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot))), "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copies_end_row() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>  // waits for this thread's copies of all rows but the last LATER
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory");
}

// Two sums at once. The warps' sums are read by every thread and added in their order, which takes fewer turns than shuffles.
template <int TEAM>
__device__ __forceinline__ float2 team_sum2(float2 v, float2* red) {
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o; o >>= 1)
        v = add2(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
    if constexpr (TEAM > 32) {
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TEAM / 32; ++w) v = add2(v, red[w]);
    }
    return v;
}
// One, the same way.
template <int TEAM>
__device__ __forceinline__ float team_sum1(float v, float* red) {
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TEAM > 32) {
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TEAM / 32; ++w) v += red[w];
    }
    return v;
}
// The larger of top and both magnitudes; a NaN stays one.
__device__ __forceinline__ float max_abs(float top, const float2& v) {
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(v.x), "f"(v.y));
    return top;
}

// Quotients v / scale by a product t with the scale's correctly rounded reciprocal, made good by its remainder (v - t scale, exact in a
// multiply-add) times the same (Markstein 1990): correctly rounded while no term leaves f32's normal numbers. (Where a last bit could
// move an 8-bit code, next to the middles of int8 and of e4m3, tried for every scale's digits: none is off.) less: minus the scale.
__device__ __forceinline__ float2 quotient2(const float2& v, const float2& inv, const float2& less) {
    const float2 t = mul2(v, inv);
    return fma2(fma2(t, less, v), inv, t);
}

// v rounded to nearest, ties to even, and saturated to +-127; a NaN is 0.
__device__ __forceinline__ int i8_code(float v) { return min(max(__float2int_rn(v), -127), 127); }
__device__ __forceinline__ uint32_t i8_pack4(int a, int b, int c, int d) {
    return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | static_cast<uint32_t>(d) << 24;
}
// store8 as int8, from values divided by their scale.
template <int TEAM, bool VEC>
__device__ __forceinline__ void store8_i8(void* p, int64_t row, int u, int me, int cols, const float (&f)[kVec]) {
    int8_t* const q = static_cast<int8_t*>(p) + row;
    if (VEC) {
        const int c = column<TEAM, VEC>(u, 0, me);
        if (c < cols)
            *reinterpret_cast<uint2*>(q + c) = make_uint2(i8_pack4(i8_code(f[0]), i8_code(f[1]), i8_code(f[2]), i8_code(f[3])),
                                                          i8_pack4(i8_code(f[4]), i8_code(f[5]), i8_code(f[6]), i8_code(f[7])));
    } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            const int c = column<TEAM, VEC>(u, j, me);
            if (c < cols) q[c] = static_cast<int8_t>(i8_code(f[j]));
        }
    }
}

// The same of numbers that round to no more than 127: 1.5 * 2^23 added, a code is the low byte of the sum.
template <int TEAM>
__device__ __forceinline__ void store8_i8_within(void* p, int64_t row, int u, int me, int cols, const float (&f)[kVec]) {
    const int c = column<TEAM, true>(u, 0, me);
    if (c >= cols) return;
    uint32_t w[kVec];
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
        const float2 v = add2(pair_of(f, i), make_float2(12582912.f, 12582912.f));
        w[2 * i] = __float_as_uint(v.x);
        w[2 * i + 1] = __float_as_uint(v.y);
    }
    uint32_t out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        out[i] = __byte_perm(__byte_perm(w[4 * i], w[4 * i + 1], 0x0040), __byte_perm(w[4 * i + 2], w[4 * i + 3], 0x0040), 0x5410);
    *reinterpret_cast<uint2*>(static_cast<int8_t*>(p) + row + c) = make_uint2(out[0], out[1]);
}

// Rows that a team reads or writes eight values at a time: 16-byte aligned (8-byte of 8-bit types). A null is.
inline bool rows_of_eights(const void* p, int64_t stride, int type) {
    const int64_t size = type == kTokF32 ? 4 : type == kTokE4M3 || type == kTokI8 ? 1 : 2, unit = size == 1 ? 8 : 16;
    return !p || (reinterpret_cast<uintptr_t>(p) % unit == 0 && stride * size % unit == 0);
}

}  // namespace
}  // namespace fxk
