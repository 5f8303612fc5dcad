// i8_linear.cuh — what the kernels of the 8-bit linear layer share.
#pragma once

#include "token.cuh"

namespace fxk {

// Rows of bytes that TMA brings: every row begins at a multiple of 16 bytes (one row alone has no stride).
inline bool tma_rows(const void* p, int64_t stride, int64_t rows) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride % 16 == 0 || rows == 1);
}

#ifdef __CUDACC__
// A result from its exact sum: the same in every kernel, so that it does not depend on the way taken. Without a bias, bias
// is -0, which changes nothing.
__device__ __forceinline__ float i8_value(int sum, float x_scale, float scale, float bias) {
    return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(sum), x_scale), scale), bias);
}
#endif

}  // namespace fxk
