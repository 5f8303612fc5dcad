// i8_linear.cuh — what the kernels of the 8-bit linear layer share.
#pragma once

#include "pairs.cuh"
#include "ptx.cuh"
#include "token.cuh"

namespace fxk {

constexpr int kI8Step = 128;  // inputs of a step: a swizzled line of shared memory a row
constexpr int kI8MaxSlots = 8;
constexpr int kI8StreamRows = 128;  // at most

// Rows of bytes that TMA brings: every row begins at a multiple of 16 bytes (one row alone has no stride).
inline bool tma_rows(const void* p, int64_t stride, int64_t rows) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride % 16 == 0 || rows == 1);
}

cudaError_t launch_i8_stream(const I8LinearArgs& a, cudaStream_t s);
cudaError_t launch_i8_pair(const I8LinearArgs& a, cudaStream_t s);
// The status words of the files' kernels, cleared.
cudaError_t i8_stream_status(uint32_t* code);
cudaError_t i8_pair_status(uint32_t* code);

#ifdef __CUDACC__
// Set by a kernel of this file's includer whose bounded wait gave up; read and cleared by take_i8_status.
static __device__ uint32_t g_i8_status;

static inline cudaError_t take_i8_status(uint32_t* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_i8_status, sizeof *code);
    const uint32_t zero = 0;
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_i8_status, &zero, sizeof zero);
    return e;
}

// Four s32 of a block of the cluster, at a shared-memory address of this one.
__device__ __forceinline__ int4 ld_cluster_s32x4(uint32_t addr, int rank) {
    int4 v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\tld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [r];\n\t}"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr), "r"(rank));
    return v;
}

// A result from its exact sum, rounded to f32: the same in every kernel, so that it does not depend on the way taken. Without a bias, bias
// is -0, which changes nothing.
__device__ __forceinline__ float i8_value(float sum, float x_scale, float scale, float bias) {
    return __fadd_rn(__fmul_rn(__fmul_rn(sum, x_scale), scale), bias);
}
__device__ __forceinline__ float2 i8_value(const float2& sum, float x_scale, const float2& scale, const float2& bias) {
    const float2 v = mul2(mul2(sum, make_float2(x_scale, x_scale)), scale);
    return make_float2(__fadd_rn(v.x, bias.x), __fadd_rn(v.y, bias.y));  // (a pair's sum may be fused with the product before it)
}
__device__ __forceinline__ float i8_value(int sum, float x_scale, float scale, float bias) {
    return i8_value(__int2float_rn(sum), x_scale, scale, bias);
}
// Four results to consecutive outputs; vec: all four are there and aligned.
__device__ __forceinline__ void i8_store4(void* y, int64_t at, int type, const float (&f)[4], bool vec, int there) {
    if (!vec) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < there) tok_store(y, at + e, type, f[e]);
    } else if (type == kTokF32) {
        *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        uint32_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (type == kTokF16) {
                const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
                w[e] = reinterpret_cast<const uint32_t&>(h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
                w[e] = reinterpret_cast<const uint32_t&>(h);
            }
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + at) = make_uint2(w[0], w[1]);
    }
}
#endif

}  // namespace fxk
