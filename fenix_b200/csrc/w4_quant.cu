// w4_quant.cu — weights to 4-bit codes with group scales (and zero points), and back.
#include "counters.hpp"
#include "token.cuh"

namespace fxk {
namespace {

constexpr int kThreads = 256;

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

// One warp per group.
__global__ void __launch_bounds__(kThreads) w4_quantize_kernel(const void* w, int w_type, int64_t w_stride, const W4Args q) {
    const int lane = threadIdx.x % 32;
    const int per_row = q.k / q.group;
    const int64_t g = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    if (g >= static_cast<int64_t>(q.n) * per_row) return;
    const int64_t base = g / per_row * w_stride + g % per_row * q.group;
    float lo = 0.f, hi = 0.f;
    for (int i = lane; i < q.group; i += 32) {
        const float v = tok_load(w, base + i, w_type);
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    for (int o = 16; o; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float scale = round_scale(q.zeros ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f), q.scale_type);
    float zero = 8.f;
    if (q.zeros) zero = scale > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, scale)), 0.f), 15.f) : 0.f;
    if (lane == 0) {
        tok_store(const_cast<void*>(q.scales), g, q.scale_type, scale);
        if (q.zeros) const_cast<uint8_t*>(q.zeros)[g] = static_cast<uint8_t>(zero);
    }
    for (int i = 2 * lane; i < q.group; i += 64) {
        const float a = code_of(tok_load(w, base + i, w_type), scale, zero);
        const float b = code_of(tok_load(w, base + i + 1, w_type), scale, zero);
        const_cast<uint8_t*>(q.codes)[(g * q.group + i) / 2] =
            static_cast<uint8_t>(static_cast<int>(a) | static_cast<int>(b) << 4);
    }
}

__global__ void __launch_bounds__(kThreads) w4_dequantize_kernel(const W4Args q, void* w, int w_type, int64_t w_stride) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 2;
    if (i >= static_cast<int64_t>(q.n) * q.k) return;
    const int64_t g = i / q.group, o = i / q.k * w_stride + i % q.k;
    const int c = q.codes[i / 2];
    const int z = q.zeros ? q.zeros[g] : 8;
    const float s = tok_load(q.scales, g, q.scale_type);
    tok_store(w, o, w_type, s * static_cast<float>((c & 15) - z));
    tok_store(w, o + 1, w_type, s * static_cast<float>((c >> 4) - z));
}

}  // namespace

cudaError_t launch_w4_quantize(const void* w, int w_type, int64_t w_stride, const W4Args& q, cudaStream_t s) {
    const int64_t groups = static_cast<int64_t>(q.n) * (q.k / q.group);
    const int64_t blocks = (groups + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    count_launch();
    w4_quantize_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(w, w_type, w_stride, q);
    return cudaGetLastError();
}

cudaError_t launch_w4_dequantize(const W4Args& q, void* w, int w_type, int64_t w_stride, cudaStream_t s) {
    const int64_t blocks = (static_cast<int64_t>(q.n) * q.k / 2 + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    count_launch();
    w4_dequantize_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(q, w, w_type, w_stride);
    return cudaGetLastError();
}

}  // namespace fxk
