// pairs.cuh — two f32 operations in one instruction. The compiler may fuse a pair's product with the pair's sum after it into one
// rounding.
#pragma once

#include <cstdint>

namespace fxk {

__device__ __forceinline__ float2 pair_of(const float* f, int i) { return make_float2(f[2 * i], f[2 * i + 1]); }
__device__ __forceinline__ void put_pair(float* f, int i, const float2& v) {
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
}
__device__ __forceinline__ uint64_t bits_of(const float2& v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 pair_of(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return pair_of(r);
}
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return pair_of(r);
}
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
    return pair_of(r);
}

}  // namespace fxk
