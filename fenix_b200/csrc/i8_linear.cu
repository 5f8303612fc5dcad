// i8_linear.cu — linear layer of 8-bit integers: which kernel a call takes, and the one that takes rows of any alignment.
//
// Sums are 32-bit integers, so every order of adding gives the same: k may be cut into ranges without changing a result.
#include "counters.hpp"
#include "i8_linear.cuh"

#include <algorithm>

namespace fxk {
namespace {

// ---- rows of any alignment -------------------------------------------------------------------------------------------
// A tile of 64 rows by 64 outputs, 64 inputs a step, on m16n8k32 MMAs: four warps of 32 by 32 each. The next step's bytes
// wait in registers while the warps multiply this one's.
constexpr int kTile = 64, kStep = 64, kPitch = kStep + 16;

// 16 bytes of a row from input k0 on, zeros past its end. Of unaligned ones the five words around them are read where all
// five lie inside the row.
__device__ __forceinline__ uint4 bytes16(const int8_t* row, int k0, int k) {
    const int8_t* const p = row + k0;
    uint32_t w[4];
    if (k0 + 16 <= k) {
        const uint32_t off = reinterpret_cast<uintptr_t>(p) & 3;
        if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) return __ldg(reinterpret_cast<const uint4*>(p));
        if (off == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (k0 >= 4 && k0 + 20 <= k) {
            const uint32_t* const q = reinterpret_cast<const uint32_t*>(p - off);
            uint32_t v = __ldg(q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t next = __ldg(q + i + 1);
                w[i] = __funnelshift_r(v, next, off * 8);
                v = next;
            }
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k0 + 4 * i + j < k) w[i] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(p + 4 * i + j))) << (8 * j);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ void __launch_bounds__(128) i8_any_kernel(const __grid_constant__ I8LinearArgs a) {
    __shared__ __align__(16) uint8_t xs[kTile * kPitch], ws[kTile * kPitch];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int64_t o0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int rm = warp / 2 * 32, om = warp % 2 * 32;  // the warp's corner in the tile
    uint4 xv[2], wv[2];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = threadIdx.x / 4 + i * 32, at = k0 + threadIdx.x % 4 * 16;
            xv[i] = wv[i] = make_uint4(0, 0, 0, 0);
            if (at < a.k && r0 + row < a.rows) xv[i] = bytes16(a.x + (r0 + row) * a.x_stride, at, a.k);
            if (at < a.k && o0 + row < a.n) wv[i] = bytes16(a.codes + (o0 + row) * a.codes_stride, at, a.k);
        }
    };
    int acc[2][4][4] = {};
    fetch(0);
    for (int k0 = 0; k0 < a.k; k0 += kStep) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int to = (threadIdx.x / 4 + i * 32) * kPitch + threadIdx.x % 4 * 16;
            *reinterpret_cast<uint4*>(xs + to) = xv[i];
            *reinterpret_cast<uint4*>(ws + to) = wv[i];
        }
        __syncthreads();
        if (k0 + kStep < a.k) fetch(k0 + kStep);
#pragma unroll
        for (int kk = 0; kk < kStep; kk += 32) {
            uint32_t af[2][4], bf[4][2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    af[m][i] = *reinterpret_cast<const uint32_t*>(xs + (rm + m * 16 + g + i % 2 * 8) * kPitch + kk + i / 2 * 16 + t * 4);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    bf[n][i] = *reinterpret_cast<const uint32_t*>(ws + (om + n * 8 + g) * kPitch + kk + i * 16 + t * 4);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                        : "+r"(acc[m][n][0]), "+r"(acc[m][n][1]), "+r"(acc[m][n][2]), "+r"(acc[m][n][3])
                        : "r"(af[m][0]), "r"(af[m][1]), "r"(af[m][2]), "r"(af[m][3]), "r"(bf[n][0]), "r"(bf[n][1]));
        }
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t row = r0 + rm + m * 16 + i * 8 + g;
            if (row >= a.rows) continue;
            const float scale = a.x_scale[a.x_scale_mode == kScaleRow ? row : 0];
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int64_t o = o0 + om + n * 8 + t * 2 + e;
                    if (o < a.n)
                        tok_store(a.y, row * a.y_stride + o, a.y_type,
                                  i8_value(acc[m][n][i * 2 + e], scale, a.scales[o], a.bias ? a.bias[o] : -0.f));
                }
        }
}

cudaError_t launch_any(const I8LinearArgs& a, cudaStream_t s) {
    constexpr int64_t kRows = int64_t{65535} * kTile;  // of a launch
    for (int64_t row = 0; row < a.rows; row += kRows) {
        I8LinearArgs part = a;
        part.rows = static_cast<int>(std::min<int64_t>(kRows, a.rows - row));
        part.x = a.x + row * a.x_stride;
        if (a.x_scale_mode == kScaleRow) part.x_scale = a.x_scale + row;
        part.y = static_cast<uint8_t*>(a.y) + row * a.y_stride * (a.y_type == kTokF32 ? 4 : 2);
        count_launch();
        i8_any_kernel<<<dim3((a.n + kTile - 1) / kTile, (part.rows + kTile - 1) / kTile), 128, 0, s>>>(part);
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_i8_linear(const I8LinearArgs& a, cudaStream_t s) {
    if (!tma_rows(a.x, a.x_stride, a.rows) || !tma_rows(a.codes, a.codes_stride, a.n)) return launch_any(a, s);
    // Few rows stream weights past them, more share tiles of 256 rows and up to 256 outputs between two SMs. The stream's blocks
    // bring every row with 128 outputs, which costs more than the pairs' fixed time once they are many (us, stream and pairs:
    // 32 x 4096 -> 14336 15.9 and 16.2, 64 rows 19.4 and 16.6; 64 x 8192 -> 8192 19.4 and 21.7, 128 rows 20.7 and 22.4, 192 rows
    // 25.8 and 22; 128 x 4096 -> 28672 45 and 29).
    const bool stream = a.rows <= 32 || (a.rows <= 128 && a.n <= sm_count() / 2 * 128);
    return stream ? launch_i8_stream(a, s) : launch_i8_pair(a, s);
}

}  // namespace fxk
