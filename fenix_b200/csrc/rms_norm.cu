// rms_norm.cu — root-mean-square norm of token rows with the residual's addition and 8-bit output.
#include "counters.hpp"
#include "token.cuh"

namespace fxk {
namespace {

constexpr int kThreads = 256;

// Sum and maximum of a value over the block; every thread gets them.
__device__ float block_sum(float v, float* red) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < kThreads / 32; ++i) v += red[i];
    return v;
}
__device__ uint32_t block_max(uint32_t v, uint32_t* red) {
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kThreads / 32; ++i) v = max(v, red[i]);
    return v;
}

// One block per row, the row's h in shared memory.
__global__ void __launch_bounds__(kThreads) rms_norm_kernel(const RmsNormArgs a) {
    extern __shared__ float h[];
    __shared__ float red[kThreads / 32];
    const int64_t row = blockIdx.x;
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        float v = tok_load(a.x, row * a.x_stride + c, a.x_type);
        if (a.residual) v += tok_load(a.residual, row * a.residual_stride + c, a.residual_type);
        h[c] = v;
        ss += v * v;
    }
    ss = block_sum(ss, red);
    float pre = 1.f;
    if (!(ss < 3.0e38f)) {  // squares past f32's range (or a NaN or infinity, which stays one): sum smaller ones
        pre = 8.2718061e-25f;  // 2^-80
        ss = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) ss += (h[c] * pre) * (h[c] * pre);
        ss = block_sum(ss, red);
    }
    const float r = rsqrtf(ss / static_cast<float>(a.cols) + a.eps * pre * pre);
    float scale = a.scale_mode == kScaleTensor ? a.scale[0] : 1.f;
    uint32_t amax = 0;  // |v| as bits: a NaN is above every number
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        if (a.sum) tok_store(a.sum, row * a.sum_stride + c, a.residual_type, h[c]);
        h[c] = h[c] * pre * r * (a.weight ? tok_load(a.weight, c, a.weight_type) : 1.f);
        amax = max(amax, __float_as_uint(h[c]) & 0x7fffffffu);
    }
    if (a.scale_mode == kScaleRow) {
        amax = block_max(amax, reinterpret_cast<uint32_t*>(red));
        amax = max(amax, __float_as_uint(1e-30f));
        scale = __uint_as_float(amax) / 448.f;
        if (threadIdx.x == 0) a.scale[row] = scale;
    }
    const float inv = 1.f / scale;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) tok_store(a.y, row * a.y_stride + c, a.y_type, h[c] * inv);
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormArgs& a, cudaStream_t s) {
    const size_t smem = static_cast<size_t>(a.cols) * sizeof(float);
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(rms_norm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kRmsMaxCols * static_cast<int>(sizeof(float)));
        if (e != cudaSuccess) return e;
    }
    count_launch();
    rms_norm_kernel<<<a.rows, kThreads, smem, s>>>(a);
    return cudaGetLastError();
}

}  // namespace fxk
