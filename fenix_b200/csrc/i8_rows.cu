// i8_rows.cu — rows to int8 codes with a scale a row (or one for the tensor), and back.
//
// Bound by memory: a value passes once (4 or 2 bytes in, one out). A team of threads holds a row in registers between its
// largest magnitude and its codes; rows past 16384 values are read twice, the second time mostly from the caches.
// Codes are those of f32's correctly rounded quotients: a product with the scale's reciprocal stands for the quotient
// unless it lies so near a half that the two might round differently; then the quotient is taken.
#include "counters.hpp"
#include "token_rows.cuh"

namespace fxk {
namespace {

// Code of x / scale. The product t = x inv is off from the rounded quotient by less than 2^-22 |t| <= 2^-14 while |t| < 256 (the
// reciprocal, the product and the quotient are rounded once each, 2^-24), so rounding it gives the quotient's code if it is
// further than 2^-13 from a half.
__device__ __forceinline__ float code_near(float x, float scale, float inv) {
    const float t = x * inv, r = rintf(t);
    if (!(fabsf(t - r) < 0.5f - 1.220703125e-4f) || !(fabsf(t) < 256.f)) return __fdiv_rn(x, scale);
    return r;
}

// The reciprocal that code_near takes; one that would be near f32's smallest values is infinite, so that every quotient is taken.
__device__ __forceinline__ float inverse(float scale) { return scale < 1e37f ? 1.f / scale : INFINITY; }

// Scale of a row from its largest magnitude's bits (a NaN is above every number).
__device__ __forceinline__ float row_scale(uint32_t top) {
    return __fdiv_rn(__uint_as_float(max(top, __float_as_uint(1e-30f))), 127.f);
}

template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM) i8_quantize_kernel(const __grid_constant__ I8RowsArgs a) {
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
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) top = max(top, __float_as_uint(f[u][j]) & 0x7fffffffu);
        scale = row_scale(team_max<TEAM>(top, red));
        if (me == 0 && cols) a.scale[row] = scale;
    } else {
        scale = a.scale[0];
    }
    const float inv = inverse(scale);
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[u][j] = code_near(f[u][j], scale, inv);
        store8_i8<TEAM, VEC>(a.codes, row * a.codes_stride, u, me, cols, f[u]);
    }
}

// A block a row, of any length.
constexpr int kWide = 1024;
template <bool VEC>
__global__ void __launch_bounds__(kWide) i8_quantize_wide_kernel(const __grid_constant__ I8RowsArgs a) {
    __shared__ uint32_t red[32];
    const int64_t row = blockIdx.x;
    const int turns = (a.cols + kWide * kVec - 1) / (kWide * kVec);
    float scale;
    if (a.scale_mode == kScaleRow) {
        uint32_t top = 0;
        for (int u = 0; u < turns; ++u) {
            float f[kVec];
            load8<kWide, VEC, false>(a.x, row * a.stride, a.type, u, threadIdx.x, a.cols, f);
#pragma unroll
            for (int j = 0; j < kVec; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
        }
        scale = row_scale(team_max<kWide>(top, red));
        if (threadIdx.x == 0) a.scale[row] = scale;
    } else {
        scale = a.scale[0];
    }
    const float inv = inverse(scale);
    for (int u = 0; u < turns; ++u) {
        float f[kVec];
        load8<kWide, VEC, false>(a.x, row * a.stride, a.type, u, threadIdx.x, a.cols, f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[j] = code_near(f[j], scale, inv);
        store8_i8<kWide, VEC>(a.codes, row * a.codes_stride, u, threadIdx.x, a.cols, f);
    }
}

// A thread takes eight codes (VEC) or one, in rows of blockIdx.y, ...
template <bool VEC>
__global__ void __launch_bounds__(256) i8_dequantize_kernel(const __grid_constant__ I8RowsArgs a) {
    constexpr int kEach = VEC ? kVec : 1;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * kEach;
    if (c >= a.cols) return;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float scale = a.scale[a.scale_mode == kScaleRow ? row : 0];
        const int8_t* const q = a.codes + row * a.codes_stride + c;
        const int64_t o = row * a.stride + c;
        if constexpr (VEC) {
            const uint2 w = *reinterpret_cast<const uint2*>(q);
            float f[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) f[j] = scale * static_cast<float>(static_cast<int8_t>((j < 4 ? w.x : w.y) >> (8 * (j % 4))));
            store8<1, true>(a.y, o, a.type, 0, 0, kVec, f);
        } else {
            tok_store(a.y, o, a.type, scale * static_cast<float>(*q));
        }
    }
}

template <int TEAM, int TURNS>
cudaError_t quantize(const I8RowsArgs& a, bool vec, cudaStream_t s) {
    constexpr int threads = TEAM <= 32 ? 128 : TEAM, per = threads / TEAM;
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + per - 1) / per);
    count_launch();
    if (vec)
        i8_quantize_kernel<TEAM, TURNS, true><<<grid, threads, 0, s>>>(a);
    else
        i8_quantize_kernel<TEAM, TURNS, false><<<grid, threads, 0, s>>>(a);
    return cudaGetLastError();
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
    if (vec)
        i8_quantize_wide_kernel<true><<<a.rows, kWide, 0, s>>>(a);
    else
        i8_quantize_wide_kernel<false><<<a.rows, kWide, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_i8_dequantize(const I8RowsArgs& a, cudaStream_t s) {
    const bool vec = both_aligned(a, a.y);
    const unsigned across = static_cast<unsigned>((a.cols + 256 * (vec ? kVec : 1) - 1) / (256 * (vec ? kVec : 1)));
    const dim3 grid(across, a.rows < 65535 ? a.rows : 65535);
    count_launch();
    if (vec)
        i8_dequantize_kernel<true><<<grid, 256, 0, s>>>(a);
    else
        i8_dequantize_kernel<false><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace fxk
