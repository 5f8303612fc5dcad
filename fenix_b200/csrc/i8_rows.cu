// i8_rows.cu — rows to int8 codes with a scale a row (or one for the tensor), and back.
//
// Bound by memory: a value passes once (4 or 2 bytes in, one out). A team of threads holds a row in registers between its
// largest magnitude and its codes; rows past 16384 values are read twice, the second time mostly from the caches.
// Codes are those of f32's correctly rounded quotients. 8192 x 8192 f32 49 us, 6.8 TB/s, and 35 back to bf16, 5.8 TB/s; bf16
// 44 us, 4.6 TB/s, where a row's load, maximum and codes follow one another in a block.
#include "counters.hpp"
#include "token_rows.cuh"

namespace fxk {
namespace {

// Code of x / scale. The product t = x inv is off from the rounded quotient by less than 2^-22 |t| <= 2^-14 while |t| < 256 (the
// reciprocal, the product and the quotient are rounded once each, 2^-24), so rounding it gives the quotient's code if it is
// further than 2^-13 from a half.
constexpr float kNearHalf = 0.5f - 1.220703125e-4f;
__device__ __forceinline__ float code_near(float x, float scale, float inv) {
    const float t = x * inv, r = rintf(t);
    if (!(fabsf(t - r) < kNearHalf) || !(fabsf(t) < 256.f)) return __fdiv_rn(x, scale);
    return r;
}

// The reciprocal that code_near takes; one that would be near f32's smallest values is infinite, so that every quotient is taken.
__device__ __forceinline__ float inverse(float scale) { return scale < 1e37f ? 1.f / scale : INFINITY; }

// Scale of a row from its largest magnitude's bits (a NaN is above every number).
__device__ __forceinline__ float row_scale(uint32_t top) {
    return __fdiv_rn(__uint_as_float(max(top, __float_as_uint(1e-30f))), 127.f);
}

// Eight codes of a row under its own scale, from whose quotients none is past 127, where no term of quotient2 falls below f32's
// normal numbers.
__device__ __forceinline__ bool has_codes8(float scale) { return scale > 1e-28f && scale < 1e37f; }
__device__ __forceinline__ uint2 codes8(const float (&x)[kVec], float scale, float inv) {
    const float2 inv2 = make_float2(inv, inv), less2 = make_float2(-scale, -scale);
    uint32_t w[kVec];
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
        const float2 q = quotient2(pair_of(x, i), inv2, less2);
        const float2 m = add2(q, make_float2(12582912.f, 12582912.f));  // 1.5 * 2^23: the sum's low byte is the code
        w[2 * i] = __float_as_uint(m.x);
        w[2 * i + 1] = __float_as_uint(m.y);
    }
    uint32_t out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        out[i] = __byte_perm(__byte_perm(w[4 * i], w[4 * i + 1], 0x0040), __byte_perm(w[4 * i + 2], w[4 * i + 3], 0x0040), 0x5410);
    return make_uint2(out[0], out[1]);
}

template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM, TEAM <= 32 ? 1 : 2048 / TEAM) i8_quantize_kernel(const __grid_constant__ I8RowsArgs a) {
    wait_for_earlier();
    let_later_begin();
    __shared__ uint32_t red[32];
    constexpr int kPer = TEAM <= 32 ? 128 / TEAM : 1;
    const int me = threadIdx.x % TEAM;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kPer + threadIdx.x / TEAM;
    const int cols = row < a.rows ? a.cols : 0;  // lanes of no row run along: the maximum is the warp's
    float f[TURNS][kVec];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) load8<TEAM, VEC, false>(a.x, row * a.stride, a.type, u, me, cols, f[u]);
    float scale;
    if (a.scale_mode == kScaleRow) {
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) top = max_abs(top, pair_of(f[u], i));
        scale = row_scale(team_max<TEAM>(__float_as_uint(top), red));
        if (me == 0 && cols) a.scale[row] = scale;
    } else {
        scale = a.scale[0];
    }
    const float inv = inverse(scale);
    const bool plain = VEC && a.scale_mode == kScaleRow && has_codes8(scale);
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        if (plain) {
            const int c = column<TEAM, true>(u, 0, me);
            if (c < cols) *reinterpret_cast<uint2*>(a.codes + row * a.codes_stride + c) = codes8(f[u], scale, inv);
            continue;
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[u][j] = code_near(f[u][j], scale, inv);
        store8_i8<TEAM, VEC>(a.codes, row * a.codes_stride, u, me, cols, f[u]);
    }
}

// A block a row, of any length.
constexpr int kWide = 1024;
template <bool VEC>
__global__ void __launch_bounds__(kWide) i8_quantize_wide_kernel(const __grid_constant__ I8RowsArgs a) {
    wait_for_earlier();
    let_later_begin();
    __shared__ uint32_t red[32];
    const int64_t row = blockIdx.x;
    const int turns = (a.cols + kWide * kVec - 1) / (kWide * kVec);
    float scale;
    if (a.scale_mode == kScaleRow) {
        float top = 0.f;
#pragma unroll 2
        for (int u = 0; u < turns; ++u) {
            float f[kVec];
            load8<kWide, VEC, false>(a.x, row * a.stride, a.type, u, threadIdx.x, a.cols, f);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) top = max_abs(top, pair_of(f, i));
        }
        scale = row_scale(team_max<kWide>(__float_as_uint(top), red));
        if (threadIdx.x == 0) a.scale[row] = scale;
    } else {
        scale = a.scale[0];
    }
    const float inv = inverse(scale);
    const bool plain = VEC && a.scale_mode == kScaleRow && has_codes8(scale);
#pragma unroll 2
    for (int u = 0; u < turns; ++u) {
        float f[kVec];
        load8<kWide, VEC, false>(a.x, row * a.stride, a.type, u, threadIdx.x, a.cols, f);
        if (plain) {
            const int c = column<kWide, true>(u, 0, threadIdx.x);
            if (c < a.cols) *reinterpret_cast<uint2*>(a.codes + row * a.codes_stride + c) = codes8(f, scale, inv);
            continue;
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[j] = code_near(f[j], scale, inv);
        store8_i8<kWide, VEC>(a.codes, row * a.codes_stride, u, threadIdx.x, a.cols, f);
    }
}

// A thread takes N codes (eight for 16-bit values, four for f32, so that a warp's store is whole lines; or one, of rows that
// are not aligned) of four rows at a time.
constexpr int kBackRows = 4;
template <int N>
__global__ void __launch_bounds__(256) i8_dequantize_kernel(const __grid_constant__ I8RowsArgs a) {
    wait_for_earlier();
    let_later_begin();
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * N;
    if (c >= a.cols) return;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.y) * kBackRows; row0 < a.rows; row0 += static_cast<int64_t>(gridDim.y) * kBackRows) {
        uint32_t w[kBackRows][2];
        float scale[kBackRows];
#pragma unroll
        for (int i = 0; i < kBackRows; ++i) {
            const int64_t row = row0 + i;
            if (row >= a.rows) break;
            scale[i] = a.scale[a.scale_mode == kScaleRow ? row : 0];
            const int8_t* const q = a.codes + row * a.codes_stride + c;
            if constexpr (N == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(q);
                w[i][0] = v.x, w[i][1] = v.y;
            } else if constexpr (N == 4) {
                w[i][0] = *reinterpret_cast<const uint32_t*>(q);
            } else {
                w[i][0] = static_cast<uint8_t>(*q);
            }
        }
#pragma unroll
        for (int i = 0; i < kBackRows; ++i) {
            const int64_t row = row0 + i, o = row * a.stride + c;
            if (row >= a.rows) break;
            if constexpr (N > 1) {
                float f[N];
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    // code + 128 under the exponent of 2^23, less that and 128
                    const uint32_t v = w[i][j / 2] ^ 0x80808080u;
                    const float2 t = add2(make_float2(__uint_as_float(__byte_perm(v, 0x4b000000u, 0x7650 + 2 * j % 4)),
                                                      __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7650 + 2 * j % 4 + 1))),
                                          make_float2(-8388736.f, -8388736.f));
                    put_pair(f, j, mul2(t, make_float2(scale[i], scale[i])));
                }
                if constexpr (N == 4)
                    *reinterpret_cast<float4*>(static_cast<float*>(a.y) + o) = make_float4(f[0], f[1], f[2], f[3]);
                else
                    store8<1, true>(a.y, o, a.type, 0, 0, kVec, f);
            } else {
                tok_store(a.y, o, a.type, scale[i] * static_cast<float>(static_cast<int8_t>(w[i][0])));
            }
        }
    }
}

template <int TEAM, int TURNS>
cudaError_t quantize(const I8RowsArgs& a, bool vec, cudaStream_t s) {
    constexpr int threads = TEAM <= 32 ? 128 : TEAM, per = threads / TEAM;
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + per - 1) / per);
    count_launch();
    return launch_early(vec ? i8_quantize_kernel<TEAM, TURNS, true> : i8_quantize_kernel<TEAM, TURNS, false>, dim3(grid), threads, 0, s, a);
}

bool both_aligned(const I8RowsArgs& a, const void* values) {
    return a.cols % kVec == 0 && rows_of_eights(values, a.stride, a.type) && rows_of_eights(a.codes, a.codes_stride, kTokI8);
}

}  // namespace

cudaError_t launch_i8_quantize(const I8RowsArgs& a, cudaStream_t s) {
    const bool vec = both_aligned(a, a.x);
    if (a.cols <= 64) return quantize<8, 1>(a, vec, s);
    if (a.cols <= 256) return quantize<32, 1>(a, vec, s);
    if (a.cols <= 512) return quantize<32, 2>(a, vec, s);
    if (a.cols <= 1024) return quantize<128, 1>(a, vec, s);
    if (a.cols <= 2048) return quantize<256, 1>(a, vec, s);
    if (a.cols <= 4096) return quantize<256, 2>(a, vec, s);
    if (a.cols <= 8192) return quantize<512, 2>(a, vec, s);
    if (a.cols <= 16384) return quantize<1024, 2>(a, vec, s);
    count_launch();
    return launch_early(vec ? i8_quantize_wide_kernel<true> : i8_quantize_wide_kernel<false>, dim3(a.rows), kWide, 0, s, a);
}

cudaError_t launch_i8_dequantize(const I8RowsArgs& a, cudaStream_t s) {
    const int n = !both_aligned(a, a.y) ? 1 : a.type == kTokF32 ? 4 : 8;
    const int tall = (a.rows + kBackRows - 1) / kBackRows;
    const dim3 grid(static_cast<unsigned>((a.cols + 256 * n - 1) / (256 * n)), tall < 65535 ? tall : 65535);
    auto* kern = n == 8 ? i8_dequantize_kernel<8> : n == 4 ? i8_dequantize_kernel<4> : i8_dequantize_kernel<1>;
    count_launch();
    return launch_early(kern, grid, 256, 0, s, a);
}

}  // namespace fxk
