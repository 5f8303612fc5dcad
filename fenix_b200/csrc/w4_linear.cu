// w4_linear.cu — linear layer with 4-bit weights and group scales.
#include "counters.hpp"
#include "token.cuh"

namespace fxk {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsAtOnce = 8;

// One warp per output and eight rows; lanes over k.
__global__ void __launch_bounds__(kThreads) w4_linear_kernel(const W4LinearArgs a) {
    const int lane = threadIdx.x % 32;
    const int o = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    if (o >= a.w.n) return;
    const int64_t per_row = a.w.k / a.w.group;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * kRowsAtOnce; r0 < a.rows;
         r0 += static_cast<int64_t>(gridDim.y) * kRowsAtOnce) {
        float acc[kRowsAtOnce] = {};
        for (int i = 2 * lane; i < a.w.k; i += 64) {
            const int64_t g = o * per_row + i / a.w.group;
            const int c = a.w.codes[(static_cast<int64_t>(o) * a.w.k + i) / 2];
            const int z = a.w.zeros ? a.w.zeros[g] : 8;
            const float s = tok_load(a.w.scales, g, a.w.scale_type);
            const float w0 = s * static_cast<float>((c & 15) - z), w1 = s * static_cast<float>((c >> 4) - z);
#pragma unroll
            for (int r = 0; r < kRowsAtOnce; ++r) {
                if (r0 + r >= a.rows) break;
                const int64_t at = (r0 + r) * a.x_stride + i;
                acc[r] += w0 * tok_load(a.x, at, a.x_type) + w1 * tok_load(a.x, at + 1, a.x_type);
            }
        }
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            if (r0 + r >= a.rows) break;
            float v = acc[r];
            for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
            if (lane == 0) {
                if (a.x_scale) v *= a.x_scale[a.x_scale_mode == kScaleRow ? r0 + r : 0];
                if (a.bias) v += a.bias[o];
                tok_store(a.y, (r0 + r) * a.y_stride + o, a.y_type, v);
            }
        }
    }
}

}  // namespace

cudaError_t launch_w4_linear(const W4LinearArgs& a, cudaStream_t s) {
    const int64_t tiles = (static_cast<int64_t>(a.rows) + kRowsAtOnce - 1) / kRowsAtOnce;
    dim3 grid((a.w.n + kThreads / 32 - 1) / (kThreads / 32), static_cast<unsigned>(tiles < 65535 ? tiles : 65535));
    count_launch();
    w4_linear_kernel<<<grid, kThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace fxk
