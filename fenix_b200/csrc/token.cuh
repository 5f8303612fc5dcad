// token.cuh — operators over token rows: RMS norm with the residual's addition and 8-bit output, the
// linear layer with 4-bit weights, the 4-bit quantiser. Types are fx_dtype's values.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace fxk {

enum TokType : int { kTokF32 = 0, kTokF16 = 1, kTokBF16 = 2, kTokE4M3 = 3 };
enum TokScale : int { kScaleNone = 0, kScaleTensor = 1, kScaleRow = 2 };

constexpr int kRmsMaxCols = 32768;

struct RmsNormArgs {
    const void* x;
    const void* residual;  // may be null
    void* sum;             // may be null
    const void* weight;    // may be null
    void* y;
    float* scale;  // read (kScaleTensor) or written (kScaleRow); null with kScaleNone
    int64_t x_stride, residual_stride, sum_stride, y_stride;
    int rows, cols;
    int x_type, residual_type, weight_type, y_type, scale_mode;
    float eps;
};
// SMs of the current device.
int sm_count();

cudaError_t launch_rms_norm(const RmsNormArgs& a, cudaStream_t s);

struct W4Args {
    const uint8_t* codes;  // [n][k / 2]
    const void* scales;    // [n][k / group]
    const uint8_t* zeros;  // [n][k / group] or null
    int n, k, group;
    int scale_type;
};
struct W4LinearArgs {
    W4Args w;
    const void* x;
    const float* x_scale;  // null with kScaleNone
    const float* bias;     // may be null
    void* y;
    int64_t x_stride, y_stride;
    int rows;
    int x_type, x_scale_mode, y_type;
    bool hold_codes;   // failure self-test only: no codes are brought, so that the waits for them run out
    uint64_t wait_ns;  // limit of each wait inside the kernel
};
cudaError_t launch_w4_linear(const W4LinearArgs& a, cudaStream_t s);
// codes, scales and zeros of w are written
cudaError_t launch_w4_quantize(const void* w, int w_type, int64_t w_stride, const W4Args& q, cudaStream_t s);
cudaError_t launch_w4_dequantize(const W4Args& q, void* w, int w_type, int64_t w_stride, cudaStream_t s);

#ifdef __CUDACC__
// f32, f16 or bf16
__device__ __forceinline__ float tok_load(const void* p, int64_t i, int type) {
    if (type == kTokF32) return static_cast<const float*>(p)[i];
    if (type == kTokF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// v rounded to nearest; f16 past its range becomes infinite
__device__ __forceinline__ void tok_store(void* p, int64_t i, int type, float v) {
    if (type == kTokF32)
        static_cast<float*>(p)[i] = v;
    else if (type == kTokF16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
// the same of a 16-bit type, one store whichever it is
__device__ __forceinline__ void tok_store16(void* p, int64_t i, int type, float v) {
    static_cast<uint16_t*>(p)[i] =
        type == kTokF16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
#endif

}  // namespace fxk
