// w4_quant.cu — weights to 4-bit codes with group scales (and zero points), and back.
//
// Bound by memory with f32 weights: a weight passes once (4 bytes against half a byte and its share of a scale; 8192 x
// 8192 in groups of 128: 47 us, 6.4 TB/s, and 54 back), with 16-bit ones by the instructions of a weight (4096 x 14336
// bf16 with zero points: 46 us, 3.2 TB/s, and 34 back, 4.3 TB/s). A team of
// threads holds a group in registers between its extremes and its codes, eight consecutive weights a thread: 16 or
// 32 bytes in, a word of codes out, the extremes by shuffles inside the warp. Codes are those of f32's correctly
// rounded quotients: a product with the scale's reciprocal stands for the quotient unless it lies so near a half
// that the two might round differently (or is not a small number); then the quotient is taken.
#include "counters.hpp"
#include "token.cuh"

#include <algorithm>
#include <type_traits>

namespace fxk {
namespace {

constexpr int kThreads = 256;
constexpr int kEight = 8;

// v rounded to the scale's type and back; past the type's range, its largest finite value.
__device__ __forceinline__ float round_scale(float v, int type) {
    if (type == kTokF16) return __half2float(__float2half_rn(fminf(v, 65504.f)));
    if (type == kTokBF16) return __bfloat162float(__float2bfloat16_rn(fminf(v, 3.3895314e38f)));
    return fminf(v, 3.4028235e38f);
}
__device__ __forceinline__ float code_of(float w, float scale, float zero) {
    const float q = scale > 0.f && w == w ? rintf(__fdiv_rn(w, scale)) + zero : zero;
    return fminf(fmaxf(q, 0.f), 15.f);
}

// Eight codes in a word. The product t = w / scale is off by less than 2^-18 while |t| < 32, so that rounding it gives
// the quotient's code if it is further than 2^-16 from a half. The magic constant puts t + zero into the low mantissa.
// TIES: 16-bit weights do lie on halves (half of the group's largest, where that is a multiple of 7 steps); of eight
// weights only those take the quotient (8192 x 8192 bf16 in groups of 128: 54 us, 60 with a quotient for each of the
// eight; f32 49 and 47).
template <bool TIES>
__device__ __forceinline__ uint32_t codes_of(const float (&w)[kEight], float scale, float inv, float zero) {
    const float magic = 12582912.f + zero, low = -zero, high = 15.f - zero;
    auto rounded = [&](float t) { return fminf(fmaxf(t, low), high) + magic; };
    auto is_near = [&](float t, float m) { return !(fabsf(t - (m - magic)) <= 0.5f - 1.52587890625e-5f); };
    uint32_t r = 0;
    bool near = false;
#pragma unroll
    for (int j = kEight - 1; j >= 0; --j) {
        const float t = w[j] * inv, m = rounded(t);
        near |= is_near(t, m);
        r = r * 16 + __float_as_uint(m);
    }
    r -= 0x4b400000u * 0x11111111u;  // the constants of the eight
    if (near) {
#pragma unroll
        for (int j = 0; j < kEight; ++j) {
            const float t = w[j] * inv;
            if (!TIES || is_near(t, rounded(t))) r = (r & ~(15u << (4 * j))) | static_cast<uint32_t>(code_of(w[j], scale, zero)) << (4 * j);
        }
    }
    return r;
}

// How eight weights are read and held: one at a time (any type), or 16 bytes at a time of one type.
enum Kind { kAny, kVecF32, kVecF16, kVecBF16 };
template <Kind KIND>
struct Eight {  // f32, or 16-bit values as they lie in memory
    float f[kEight];
    __device__ __forceinline__ void load(const void* p, int64_t i, int type) {
        if (KIND == kVecF32) {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
            const float4 a = __ldcs(q), b = __ldcs(q + 1);
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < kEight; ++j) f[j] = tok_load(p, i + j, type);
        }
    }
    __device__ __forceinline__ void extremes(float& lo, float& hi) const {
#pragma unroll
        for (int j = 0; j < kEight; ++j) {
            lo = fminf(lo, f[j]);
            hi = fmaxf(hi, f[j]);
        }
    }
    __device__ __forceinline__ void values(float (&v)[kEight]) const {
#pragma unroll
        for (int j = 0; j < kEight; ++j) v[j] = f[j];
    }
};
template <class T2>
struct Eight16 {
    uint4 raw;
    __device__ __forceinline__ static float2 pair(uint32_t w) {
        if constexpr (std::is_same_v<T2, __half2>)
            return __half22float2(reinterpret_cast<const __half2&>(w));
        else
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    __device__ __forceinline__ void load(const void* p, int64_t i, int) { raw = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i)); }
    __device__ __forceinline__ void extremes(float& lo, float& hi) const {  // two at a time; a NaN loses against a number
        const T2* const v = reinterpret_cast<const T2*>(&raw);
        const T2 l = __hmin2(__hmin2(v[0], v[1]), __hmin2(v[2], v[3])), h = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
        const float2 a = pair(reinterpret_cast<const uint32_t&>(l)), b = pair(reinterpret_cast<const uint32_t&>(h));
        lo = fminf(lo, fminf(a.x, a.y));
        hi = fmaxf(hi, fmaxf(b.x, b.y));
    }
    __device__ __forceinline__ void values(float (&v)[kEight]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = pair(w[j]);
            v[2 * j] = t.x;
            v[2 * j + 1] = t.y;
        }
    }
};
template <>
struct Eight<kVecF16> : Eight16<__half2> {};
template <>
struct Eight<kVecBF16> : Eight16<__nv_bfloat162> {};

// TEAM lanes of a warp per group (1: groups of 32, ..., 32: any), HOLD times eight weights a lane in registers; a
// longer group is read a second time for its codes.
template <int TEAM, int HOLD, Kind KIND>
__global__ void __launch_bounds__(kThreads) w4_quantize_kernel(const void* __restrict__ w, int w_type, int64_t w_stride, const W4Args q) {
    const int me = threadIdx.x % TEAM;
    const uint32_t per_row = q.k / q.group, g32 = blockIdx.x * (kThreads / TEAM) + threadIdx.x / TEAM;  // below 2^31: the launcher's rows
    const int64_t g = g32;
    const bool on = g32 < q.n * per_row;  // lanes of no group run along: the shuffles are the warp's
    const int64_t base = on ? static_cast<int64_t>(g32 / per_row) * w_stride + g32 % per_row * static_cast<int64_t>(q.group) : 0;
    const int eights = on ? q.group / kEight : 0;
    Eight<KIND> f[HOLD];
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (h * TEAM + me < eights) f[h].load(w, base + (h * TEAM + me) * kEight, w_type);
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (h * TEAM + me < eights) f[h].extremes(lo, hi);
    for (int e = HOLD * TEAM + me; e < eights; e += TEAM) {
        Eight<KIND> t;
        t.load(w, base + static_cast<int64_t>(e) * kEight, w_type);
        t.extremes(lo, hi);
    }
#pragma unroll
    for (int o = TEAM / 2; o; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float range = q.zeros ? hi - lo : fmaxf(hi, -lo), steps = q.zeros ? 15.f : 7.f;
    if (range == INFINITY && q.zeros) range = 0.5f * hi - 0.5f * lo, steps = 7.5f;  // past f32's largest value: halves
    const float scale = round_scale(__fdiv_rn(range, steps), q.scale_type);
    float zero = 8.f;
    if (q.zeros) zero = scale > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, scale)), 0.f), 15.f) : 0.f;
    if (on && me == 0) {
        tok_store(const_cast<void*>(q.scales), g, q.scale_type, scale);
        if (q.zeros) const_cast<uint8_t*>(q.zeros)[g] = static_cast<uint8_t>(zero);
    }
    uint32_t* const codes = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(q.codes)) + g * (q.group / kEight);
    const float inv = 1.f / scale;
    auto put = [&](int e, const Eight<KIND>& t) {
        float v[kEight];
        t.values(v);
        codes[e] = codes_of<KIND == kVecF16 || KIND == kVecBF16>(v, scale, inv, zero);
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (h * TEAM + me < eights) put(h * TEAM + me, f[h]);
    for (int e = HOLD * TEAM + me; e < eights; e += TEAM) {
        Eight<KIND> t;
        t.load(w, base + static_cast<int64_t>(e) * kEight, w_type);
        put(e, t);
    }
}

// A thread makes PIECES times N consecutive values (16 bytes of them where VEC), pieces kThreads apart. A code is or'ed
// into the mantissa of 2^23.
template <bool VEC, int N, int PIECES>
__global__ void __launch_bounds__(kThreads) w4_dequantize_kernel(const W4Args q, void* __restrict__ w, int w_type, int64_t w_stride, int row0) {
    const int row = row0 + blockIdx.y, pieces = q.k / N;  // of the row
    const float inv = __frcp_rn(static_cast<float>(q.group / N));
    const uint8_t* const codes = q.codes + static_cast<int64_t>(row) * (q.k / 2);
    const int64_t g0 = static_cast<int64_t>(row) * (q.k / q.group);
    uint32_t c[PIECES];
    float s[PIECES], off[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int e = (blockIdx.x * PIECES + i) * kThreads + threadIdx.x;
        if (e >= pieces) continue;
        if constexpr (N == 8)
            c[i] = __ldcs(reinterpret_cast<const uint32_t*>(codes) + e);
        else
            c[i] = __ldcs(reinterpret_cast<const uint16_t*>(codes) + e);
        const int64_t g = g0 + static_cast<int>((static_cast<float>(e) + 0.5f) * inv);  // exact while e < 2^22, as k < 2^24
        s[i] = tok_load(q.scales, g, q.scale_type);
        off[i] = 8388608.f + (q.zeros ? static_cast<float>(__ldg(q.zeros + g)) : 8.f);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int e = (blockIdx.x * PIECES + i) * kThreads + threadIdx.x;
        if (e >= pieces) continue;
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = s[i] * (__uint_as_float((c[i] >> (4 * j) & 15u) | 0x4b000000u) - off[i]);
        const int64_t o = row * w_stride + e * N;
        if constexpr (VEC && N == 4) {
            __stcs(reinterpret_cast<float4*>(static_cast<float*>(w) + o), make_float4(f[0], f[1], f[2], f[3]));
        } else if constexpr (VEC) {
            uint32_t r[4];
            if (w_type == kTokF16) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
                    r[j] = reinterpret_cast<const uint32_t&>(h);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                    r[j] = reinterpret_cast<const uint32_t&>(h);
                }
            }
            __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(w) + o), make_uint4(r[0], r[1], r[2], r[3]));
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) tok_store(w, o + j, w_type, f[j]);
        }
    }
}

bool aligned_rows(const void* p, int64_t stride, int type) {
    const int64_t size = type == kTokF32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

template <int TEAM, int HOLD>
cudaError_t quantize(const void* w, int w_type, int64_t w_stride, const W4Args& q, cudaStream_t s) {
    const int64_t per_row = q.k / q.group, w_size = w_type == kTokF32 ? 4 : 2, s_size = q.scale_type == kTokF32 ? 4 : 2;
    const int64_t most = std::max<int64_t>((int64_t{1} << 30) / per_row, 1);  // rows of a launch
    for (int64_t row = 0; row < q.n; row += most) {
        W4Args part = q;
        part.n = static_cast<int>(std::min<int64_t>(most, q.n - row));
        part.codes = q.codes + row * (q.k / 2);
        part.scales = static_cast<const uint8_t*>(q.scales) + row * per_row * s_size;
        if (q.zeros) part.zeros = q.zeros + row * per_row;
        const void* const from = static_cast<const uint8_t*>(w) + row * w_stride * w_size;
        const unsigned blocks = static_cast<unsigned>((part.n * per_row * TEAM + kThreads - 1) / kThreads);
        count_launch();
        auto* kern = !aligned_rows(w, w_stride, w_type) ? w4_quantize_kernel<TEAM, HOLD, kAny>
                     : w_type == kTokF32                ? w4_quantize_kernel<TEAM, HOLD, kVecF32>
                     : w_type == kTokF16                ? w4_quantize_kernel<TEAM, HOLD, kVecF16>
                                                        : w4_quantize_kernel<TEAM, HOLD, kVecBF16>;
        kern<<<blocks, kThreads, 0, s>>>(from, w_type, w_stride, part);
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_w4_quantize(const void* w, int w_type, int64_t w_stride, const W4Args& q, cudaStream_t s) {
    // 32 weights a thread share what is done once a group (8192 x 8192 f32 in groups of 128: 47 us, 83 with 8 a thread);
    // a matrix that leaves SMs idle that way takes 8 a thread (1003 x 1088 bf16 in groups of 32: 3.1 us, 5.2 with 32)
    const bool small = static_cast<int64_t>(q.n) * q.k < int64_t{sm_count()} * 1024 * 32;
    if (q.group == 32) return small ? quantize<4, 1>(w, w_type, w_stride, q, s) : quantize<1, 4>(w, w_type, w_stride, q, s);
    if (q.group == 64) return small ? quantize<8, 1>(w, w_type, w_stride, q, s) : quantize<2, 4>(w, w_type, w_stride, q, s);
    if (q.group == 128) return small ? quantize<16, 1>(w, w_type, w_stride, q, s) : quantize<4, 4>(w, w_type, w_stride, q, s);
    if (q.group == 256 && !small) return quantize<8, 4>(w, w_type, w_stride, q, s);
    return quantize<32, 4>(w, w_type, w_stride, q, s);
}

cudaError_t launch_w4_dequantize(const W4Args& q, void* w, int w_type, int64_t w_stride, cudaStream_t s) {
    constexpr int kRows = 65535;  // of a launch
    // A store is 16 bytes a thread and whole lines a warp: four codes of f32 values (8192 x 8192: 54 us; 60 with eight
    // codes, whose two stores write half of every sector each), eight of 16-bit ones; four pieces a thread
    const int n = w_type == kTokF32 ? 4 : 8;
    const bool vec = aligned_rows(w, w_stride, w_type);
    const unsigned across = (q.k / n + kThreads * 4 - 1) / (kThreads * 4);
    for (int row0 = 0; row0 < q.n; row0 += kRows) {
        const dim3 grid(across, static_cast<unsigned>(q.n - row0 < kRows ? q.n - row0 : kRows));
        auto* kern = n == 4 ? (vec ? w4_dequantize_kernel<true, 4, 4> : w4_dequantize_kernel<false, 4, 4>)
                            : (vec ? w4_dequantize_kernel<true, 8, 4> : w4_dequantize_kernel<false, 8, 4>);
        count_launch();
        kern<<<grid, kThreads, 0, s>>>(q, w, w_type, w_stride, row0);
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace fxk
