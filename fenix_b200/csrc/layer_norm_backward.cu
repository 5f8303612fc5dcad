// layer_norm_backward.cu — the layer norm's backward pass: the rows' gradient, and the sums over rows that are the
// gradients of weight and bias.
//
// With z = (h - mean) rstd and g = dy weight a row's gradient needs two sums, of g and of g z:
//   dx = (g - sum(g) / n - z sum(g z) / n) rstd + dsum,   dweight = sum over rows of dy z,   dbias = sum over rows of dy
// Bound by memory: dy, h, dsum and dx pass once. Blocks stay and walk over the rows; a thread holds the same columns of every
// row, so the sums over rows stay in its registers until its block's last row, and leave as one line of the workspace a
// block, which a second kernel adds up in a fixed order.
// Rows past 8192 columns would not leave room for those sums in registers: there the rows' gradient is a kernel of its own,
// which reads a row twice (the second time from the caches), and the sums over rows another.
#include "counters.hpp"
#include "token_rows.cuh"

#include <algorithm>
#include <atomic>

namespace fxk {
namespace {

constexpr int kFusedCols = 8192;

// TEAM threads a row, TURNS times eight columns each.
template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM) layer_norm_backward_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    constexpr int kThreads = TEAM <= 32 ? 128 : TEAM, kPer = kThreads / TEAM;
    __shared__ float2 red[2][32];
    extern __shared__ float joined[];  // [2][cols]: the sums of a block of several teams
    const int me = threadIdx.x % TEAM;
    const float inv_n = 1.f / static_cast<float>(a.cols);
    float dw[TURNS][kVec] = {}, db[TURNS][kVec] = {};
    int turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kPer;
    for (int64_t lead = static_cast<int64_t>(blockIdx.x) * kPer; lead < a.rows; lead += step, turn ^= 1) {
        const int64_t row = lead + threadIdx.x / TEAM;
        const int cols = row < a.rows ? a.cols : 0;  // lanes of no row run along: the sums are the warp's
        float g[TURNS][kVec], z[TURNS][kVec];
        float mean = 0.f, rstd = 0.f;
        if (cols) mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int u = 0; u < TURNS; ++u) load8<TEAM, VEC, false>(a.dy, row * a.dy_stride, a.dy_type, u, me, cols, g[u]);
#pragma unroll
        for (int u = 0; u < TURNS; ++u) load8<TEAM, VEC, false>(a.h, row * a.h_stride, a.h_type, u, me, cols, z[u]);
        float2 sums = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            float w[kVec];
            if (a.weight) load8<TEAM, VEC, true>(a.weight, 0, a.weight_type, u, me, a.cols, w);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                z[u][j] = column<TEAM, VEC>(u, VEC ? 0 : j, me) < cols ? (z[u][j] - mean) * rstd : 0.f;
                dw[u][j] = fmaf(g[u][j], z[u][j], dw[u][j]);
                db[u][j] += g[u][j];
                if (a.weight) g[u][j] *= w[j];
                sums.x += g[u][j];
                sums.y = fmaf(g[u][j], z[u][j], sums.y);
            }
        }
        sums = team_sum2<TEAM>(sums, red[turn]);
        sums.x *= inv_n;
        sums.y *= inv_n;
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) g[u][j] = (g[u][j] - fmaf(z[u][j], sums.y, sums.x)) * rstd;
            if (a.dsum) {
                float d[kVec];
                load8<TEAM, VEC, false>(a.dsum, row * a.dsum_stride, a.dx_type, u, me, cols, d);
#pragma unroll
                for (int j = 0; j < kVec; ++j) g[u][j] += d[j];
            }
            store8<TEAM, VEC>(a.dx, row * a.dx_stride, a.dx_type, u, me, cols, g[u]);
        }
    }
    if (!a.work) return;
    float* const mine = a.work + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    if constexpr (kPer == 1) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            store8<TEAM, VEC>(mine, 0, kTokF32, u, me, a.cols, dw[u]);
            store8<TEAM, VEC>(mine, a.cols, kTokF32, u, me, a.cols, db[u]);
        }
    } else {
        // the teams of a warp by shuffles, then warp after warp
#pragma unroll
        for (int o = TEAM; o < 32; o <<= 1)
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    dw[u][j] += __shfl_xor_sync(0xffffffffu, dw[u][j], o);
                    db[u][j] += __shfl_xor_sync(0xffffffffu, db[u][j], o);
                }
        for (int w = 0; w < kThreads / 32; ++w) {
            if (threadIdx.x / 32 == w && threadIdx.x % 32 < TEAM) {
#pragma unroll
                for (int u = 0; u < TURNS; ++u)
#pragma unroll
                    for (int j = 0; j < kVec; ++j) {
                        const int c = column<TEAM, VEC>(u, VEC ? 0 : j, me) + (VEC ? j : 0);
                        if (c < a.cols) {
                            joined[c] = w ? joined[c] + dw[u][j] : dw[u][j];
                            joined[a.cols + c] = w ? joined[a.cols + c] + db[u][j] : db[u][j];
                        }
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * a.cols; c += kThreads) mine[c] = joined[c];
    }
}

// A block a row, of any length: its values are read twice.
constexpr int kWideThreads = 512;
__global__ void __launch_bounds__(kWideThreads) layer_norm_backward_wide_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    __shared__ float2 red[32];
    const int64_t row = blockIdx.x;
    const float mean = a.mean[row], rstd = a.rstd[row], inv_n = 1.f / static_cast<float>(a.cols);
    auto at = [&](int c, float& g, float& z) {
        g = tok_load(a.dy, row * a.dy_stride + c, a.dy_type);
        if (a.weight) g *= tok_load(a.weight, c, a.weight_type);
        z = (tok_load(a.h, row * a.h_stride + c, a.h_type) - mean) * rstd;
    };
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
        float g, z;
        at(c, g, z);
        sums.x += g;
        sums.y = fmaf(g, z, sums.y);
    }
    sums = team_sum2<kWideThreads>(sums, red);
    sums.x *= inv_n;
    sums.y *= inv_n;
#pragma unroll 8
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
        float g, z;
        at(c, g, z);
        g = (g - fmaf(z, sums.y, sums.x)) * rstd;
        if (a.dsum) g += tok_load(a.dsum, row * a.dsum_stride + c, a.dx_type);
        tok_store(a.dx, row * a.dx_stride + c, a.dx_type, g);
    }
}

// Sums over rows alone: a block takes 256 columns and every gridDim.y-th row.
__global__ void __launch_bounds__(256) layer_norm_sums_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    float dw = 0.f, db = 0.f;
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = tok_load(a.dy, row * a.dy_stride + c, a.dy_type);
        dw = fmaf(g, (tok_load(a.h, row * a.h_stride + c, a.h_type) - a.mean[row]) * a.rstd[row], dw);
        db += g;
    }
    float* const mine = a.work + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
    mine[c] = dw;
    mine[a.cols + c] = db;
}

// The lines of the workspace added up: 32 columns a block, eight warps that take every eighth line.
__global__ void __launch_bounds__(256) layer_norm_join_kernel(const float* __restrict__ work, int lines, int cols, float* dweight,
                                                             float* dbias, bool accumulate) {
    __shared__ float part[8][33];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;  // of dweight and dbias in a row
    const int warp = threadIdx.x / 32;
    float s = 0.f;
    if (c < 2 * cols)
#pragma unroll 8
        for (int i = warp; i < lines; i += 8) s += work[static_cast<int64_t>(i) * 2 * cols + c];
    part[warp][threadIdx.x % 32] = s;
    __syncthreads();
    if (warp || c >= 2 * cols) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
    float* const out = c < cols ? dweight : dbias;
    const int64_t o = c < cols ? c : c - cols;
    if (out) out[o] = accumulate ? out[o] + s : s;
}

template <int TEAM, int TURNS, bool VEC>
cudaError_t launch(const LayerNormBackwardArgs& a, int& lines, cudaStream_t s) {
    auto* kern = layer_norm_backward_kernel<TEAM, TURNS, VEC>;
    constexpr int threads = TEAM <= 32 ? 128 : TEAM, per = threads / TEAM;
    const size_t joined = per > 1 ? size_t{8} * a.cols : 0;  // at most 8 KB
    static std::atomic<int> known;
    int resident = known.load(std::memory_order_relaxed);
    if (!resident) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kern, threads, per > 1 ? 8192 : 0);
        if (e != cudaSuccess) return e;
        known.store(resident, std::memory_order_relaxed);
    }
    const int64_t need = (static_cast<int64_t>(a.rows) + per - 1) / per, fit = static_cast<int64_t>(sm_count()) * resident;
    lines = static_cast<int>(std::min({need, fit, layer_norm_backward_blocks(a.rows, a.cols)}));
    count_launch();
    kern<<<static_cast<unsigned>(lines), threads, joined, s>>>(a);
    return cudaGetLastError();
}
template <int TEAM, int TURNS>
cudaError_t launch(const LayerNormBackwardArgs& a, bool vec, int& lines, cudaStream_t s) {
    return vec ? launch<TEAM, TURNS, true>(a, lines, s) : launch<TEAM, TURNS, false>(a, lines, s);
}

}  // namespace

int64_t layer_norm_backward_blocks(int64_t rows, int64_t cols) {
    return std::min<int64_t>(rows, cols <= 1024 ? 1184 : cols <= 4096 ? 592 : 296);
}

cudaError_t launch_layer_norm_backward(const LayerNormBackwardArgs& a, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    if (a.rows == 0) {
        if (a.accumulate) return e;
        if (a.dweight) e = cudaMemsetAsync(a.dweight, 0, size_t{4} * a.cols, s);
        if (a.dbias && e == cudaSuccess) e = cudaMemsetAsync(a.dbias, 0, size_t{4} * a.cols, s);
        return e;
    }
    int lines = 0;
    if (a.cols > kFusedCols || !a.dx) {
        if (a.work) {
            lines = static_cast<int>(std::min<int64_t>(layer_norm_backward_blocks(a.rows, a.cols), (a.rows + 7) / 8));
            count_launch();
            layer_norm_sums_kernel<<<dim3((a.cols + 255) / 256, lines), 256, 0, s>>>(a);
            e = cudaGetLastError();
        }
        if (a.dx && e == cudaSuccess) {  // after the sums: dx may take its place over dy or h
            count_launch();
            layer_norm_backward_wide_kernel<<<a.rows, kWideThreads, 0, s>>>(a);
            e = cudaGetLastError();
        }
    } else {
        const bool vec = a.cols % kVec == 0 && rows_of_eights(a.dy, a.dy_stride, a.dy_type) &&
                         rows_of_eights(a.h, a.h_stride, a.h_type) && rows_of_eights(a.weight, 0, a.weight_type) &&
                         rows_of_eights(a.dsum, a.dsum_stride, a.dx_type) && rows_of_eights(a.dx, a.dx_stride, a.dx_type);
        if (a.cols <= 64)
            e = launch<8, 1>(a, vec, lines, s);
        else if (a.cols <= 256)
            e = launch<32, 1>(a, vec, lines, s);
        else if (a.cols <= 512)
            e = launch<32, 2>(a, vec, lines, s);
        else if (a.cols <= 1024)
            e = launch<128, 1>(a, vec, lines, s);
        else if (a.cols <= 2048)
            e = launch<256, 1>(a, vec, lines, s);
        else if (a.cols <= 4096)
            e = launch<512, 1>(a, vec, lines, s);
        else if (a.cols <= 5120)
            e = launch<640, 1>(a, vec, lines, s);
        else if (a.cols <= 6144)
            e = launch<768, 1>(a, vec, lines, s);
        else
            e = launch<1024, 1>(a, vec, lines, s);
    }
    if (e != cudaSuccess || !a.work) return e;
    count_launch();
    layer_norm_join_kernel<<<(2 * a.cols + 31) / 32, 256, 0, s>>>(a.work, lines, a.cols, a.dweight, a.dbias, a.accumulate);
    return cudaGetLastError();
}

}  // namespace fxk
