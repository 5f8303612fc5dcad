// i8_linear.cu — linear layer of 8-bit integers: which kernel a call takes, and the one that takes rows of any alignment.
//
// Sums are 32-bit integers, so every order of adding gives the same: k may be cut into ranges without changing a result.
#include "counters.hpp"
#include "i8_linear.cuh"

#include <algorithm>

namespace fxk {
namespace {

// ---- rows of any alignment -------------------------------------------------------------------------------------------
// A tile of 128 rows by 128 outputs, 64 inputs a step, on m16n8k32 MMAs: eight warps of 64 by 32 each. The next step's bytes
// wait in registers while the warps multiply this one's. Bound by the bytes' way through registers (1003 x 4705 -> 5003 in
// packed rows: 280 us, 422 with a piece after the other).
constexpr int kTile = 128, kStep = 64, kPitch = kStep + 16, kPieces = kTile * kStep / 16 / 256;

// 16 bytes of a row from input k0 on, zeros past its end, one by one.
__device__ __forceinline__ uint4 bytes16(const int8_t* row, int k0, int k) {
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k0 + i < k) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(row + k0 + i))) << (8 * (i % 4));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four 8 x 16-byte matrices, a row's address a lane.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const uint8_t* at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(at))
                 : "memory");
}

// The blocks of a cluster share a tile, steps_each steps of the inputs each; alone with split 1.
__global__ void __launch_bounds__(256) i8_any_kernel(const __grid_constant__ I8LinearArgs a, int split, int steps_each) {
    extern __shared__ __align__(16) int partial[];  // [row][output]: a cluster's sums
    __shared__ __align__(16) uint8_t xs[kTile * kPitch], ws[kTile * kPitch];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int rank = split > 1 ? static_cast<int>(blockIdx.x) % split : 0;
    const int64_t o0 = static_cast<int64_t>(blockIdx.x) / split * kTile;
    const int k_begin = rank * steps_each * kStep, k_end = min(a.k, k_begin + steps_each * kStep);  // not empty: the launcher's split
    const int rm = warp / 4 * 64, om = warp % 4 * 32;  // the warp's corner in the tile
    // a piece's 16 bytes are in the five words around them; at the ends of the rows they are put together, in the first four
    uint32_t raw[2][kPieces][5];
    bool inside = false;
    auto piece = [&](int i, int k0, int which) {  // its address, or null where there is no such row
        const int64_t row = threadIdx.x / 4 + i * 64;
        if (which ? o0 + row >= a.n : r0 + row >= a.rows) return static_cast<const int8_t*>(nullptr);
        return (which ? a.codes + (o0 + row) * a.codes_stride : a.x + (r0 + row) * a.x_stride) + k0 + threadIdx.x % 4 * 16;
    };
    auto fetch = [&](int k0) {
        inside = k0 >= 4 && k0 + kStep + 4 <= a.k;
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int8_t* const p = piece(i, k0, which);
                const int at = k0 + threadIdx.x % 4 * 16;
                if (!p) {
#pragma unroll
                    for (int e = 0; e < 5; ++e) raw[which][i][e] = 0;
                } else if (inside) {
                    const uint32_t* const q = reinterpret_cast<const uint32_t*>(p - (reinterpret_cast<uintptr_t>(p) & 3));
#pragma unroll
                    for (int e = 0; e < 5; ++e) raw[which][i][e] = __ldg(q + e);
                } else {
                    const uint4 v = at < a.k ? bytes16(p - at, at, a.k) : make_uint4(0, 0, 0, 0);
                    raw[which][i][0] = v.x, raw[which][i][1] = v.y, raw[which][i][2] = v.z, raw[which][i][3] = v.w, raw[which][i][4] = 0;
                }
            }
    };
    int acc[4][4][4] = {};
    fetch(k_begin);
    for (int k0 = k_begin; k0 < k_end; k0 += kStep) {
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint32_t shift = inside ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(piece(i, k0, which)) & 3) * 8 : 0;
                const uint32_t* const w = raw[which][i];
                *reinterpret_cast<uint4*>((which ? ws : xs) + (threadIdx.x / 4 + i * 64) * kPitch + threadIdx.x % 4 * 16) =
                    make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift), __funnelshift_r(w[2], w[3], shift),
                               __funnelshift_r(w[3], w[4], shift));
            }
        __syncthreads();
        if (k0 + kStep < k_end) fetch(k0 + kStep);
#pragma unroll
        for (int kk = 0; kk < kStep; kk += 32) {
            uint32_t af[4][4], bf[2][4];
            // lanes 0..7 address rows 0..7 of the first matrix, and so on: rows 0..7 and 8..15, then both 16 inputs on
#pragma unroll
            for (int m = 0; m < 4; ++m) ldmatrix4(af[m], xs + (rm + m * 16 + lane % 16) * kPitch + kk + lane / 16 * 16);
            // outputs 0..7 and their inputs 16 on, then outputs 8..15
#pragma unroll
            for (int n = 0; n < 2; ++n) ldmatrix4(bf[n], ws + (om + n * 16 + lane / 16 * 8 + lane % 8) * kPitch + kk + lane / 8 % 2 * 16);
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                        : "+r"(acc[m][n][0]), "+r"(acc[m][n][1]), "+r"(acc[m][n][2]), "+r"(acc[m][n][3])
                        : "r"(af[m][0]), "r"(af[m][1]), "r"(af[m][2]), "r"(af[m][3]), "r"(bf[n / 2][n % 2 * 2]), "r"(bf[n / 2][n % 2 * 2 + 1]));
        }
        __syncthreads();
    }
    if (split > 1) {  // each block adds up a share of the tile over the cluster
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    *reinterpret_cast<int2*>(partial + (rm + m * 16 + i * 8 + g) * kTile + om + n * 8 + t * 2) =
                        make_int2(acc[m][n][2 * i], acc[m][n][2 * i + 1]);
        cluster_sync();
        const int rows = static_cast<int>(min(static_cast<int64_t>(kTile), a.rows - r0)), all = rows * (kTile / 4);
        const int share = (all + split - 1) / split, end = min(all, (rank + 1) * share);
        for (int i = rank * share + threadIdx.x; i < end; i += 256) {
            int sum[4] = {};
            for (int p = 0; p < split; ++p) {
                const int4 v = ld_cluster_s32x4(smem_u32(partial) + i * 16, p);
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            }
            const int64_t row = r0 + i / (kTile / 4), o = o0 + i % (kTile / 4) * 4;
            const float scale = a.x_scale[a.x_scale_mode == kScaleRow ? row : 0];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (o + e < a.n)
                    tok_store(a.y, row * a.y_stride + o + e, a.y_type, i8_value(sum[e], scale, a.scales[o + e], a.bias ? a.bias[o + e] : -0.f));
        }
        cluster_sync();  // no block's shared memory ends while another reads it
        return;
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
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
    constexpr int kBytes = kTile * kTile * 4;
    cudaError_t e = cudaFuncSetAttribute(i8_any_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return e;
    for (int64_t row = 0; row < a.rows; row += kRows) {
        I8LinearArgs part = a;
        part.rows = static_cast<int>(std::min<int64_t>(kRows, a.rows - row));
        part.x = a.x + row * a.x_stride;
        if (a.x_scale_mode == kScaleRow) part.x_scale = a.x_scale + row;
        part.y = static_cast<uint8_t*>(a.y) + row * a.y_stride * (a.y_type == kTokF32 ? 4 : 2);
        // few tiles: clusters of as many blocks as fill the GPU once share one (1 x 4097 -> 4096 81 us without)
        const int64_t across = (a.n + kTile - 1) / kTile, down = (part.rows + kTile - 1) / kTile;
        const int steps = (a.k + kStep - 1) / kStep;
        int split = static_cast<int>(std::max<int64_t>(std::min<int64_t>({sm_count() / (across * down), 8, steps / 2}), 1));
        const int steps_each = (steps + split - 1) / split;
        split = (steps + steps_each - 1) / steps_each;  // no block without a step
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(across * split), static_cast<unsigned>(down));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = split > 1 ? kBytes : 0;
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = split;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = split > 1 ? 1 : 0;
        count_launch();
        e = cudaLaunchKernelEx(&cfg, i8_any_kernel, part, split, steps_each);
        if (e == cudaSuccess) e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_i8_linear(const I8LinearArgs& a, cudaStream_t s) {
    if (!tma_rows(a.x, a.x_stride, a.rows) || !tma_rows(a.codes, a.codes_stride, a.n)) return launch_any(a, s);
    // Few rows have the weights stream past them, more share tiles of 256 rows and up to 256 outputs between two SMs. The stream's blocks
    // bring every row with 128 outputs, which costs more than the pairs' fixed time once they are many (us, stream and pairs:
    // 32 x 4096 -> 14336 15.9 and 16.2, 64 rows 19.4 and 16.6; 64 x 8192 -> 8192 19.4 and 21.7, 128 rows 20.7 and 22.4, 192 rows
    // 25.8 and 22; 128 x 4096 -> 28672 45 and 29).
    const bool stream = a.rows <= 32 || (a.rows <= kI8StreamRows && a.n <= sm_count() / 2 * 128);
    return stream ? launch_i8_stream(a, s) : launch_i8_pair(a, s);
}

}  // namespace fxk
