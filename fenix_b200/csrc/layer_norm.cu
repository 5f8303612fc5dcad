// layer_norm.cu — layer norm of token rows with the residual's addition, the rows' statistics and 8-bit output.
//
// Bound by memory, as the RMS norm: x, residual, sum and y pass once, a row stays in the registers of its team of threads
// between the looks at it (its mean, its squares about it, its largest magnitude where it gets a scale, its output), blocks
// stay and walk over many rows with the next row on its way.
// The variance is the mean square about the mean, not a difference of two sums, so that rows far from zero keep theirs:
// t = h - mean is exact or rounded once, and the sum of the t, taken with that of their squares, gives what the mean
// itself was off by.
#include "counters.hpp"
#include "token_rows.cuh"

#include <atomic>

namespace fxk {
namespace {

struct Red {  // of a block that is one team: a row's sums, one of each look
    float2 pair[2][32];
    float sum[2][32];
    uint32_t top[32];
};

// From a row's h on; cols 0: no row, nothing is stored. red: no thread of the team still reads it.
template <int TEAM, int TURNS, bool VEC>
__device__ __forceinline__ void finish_row(const LayerNormArgs& a, int64_t row, int me, int cols, float (&h)[TURNS][kVec],
                                           Red& red) {
    const float n = static_cast<float>(a.cols);
    float mean, off, var, pre = 1.f;
    bool past;
    auto look = [&](int turn) {
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) s += h[u][j];  // columns past the row are 0
        s = team_sum<TEAM>(s, red.sum[turn]);
        mean = s / n;
        float2 q = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float t = column<TEAM, VEC>(u, VEC ? 0 : j, me) < a.cols ? h[u][j] - mean : 0.f;
                q.x += t;
                q.y = fmaf(t, t, q.y);
            }
        q = team_sum2<TEAM>(q, red.pair[turn]);
        off = q.x / n;
        var = fmaxf(q.y / n - off * off, 0.f);  // a NaN is found in past
        past = !(fabsf(s) < 3.0e38f && q.y + a.eps < 3.0e38f);
        if (q.y != q.y) var = q.y;
    };
    look(0);
    // sums past f32's range, or a NaN or infinity, which stays one: sum smaller ones
    if (TEAM < 32 ? __any_sync(0xffffffffu, past) : past) {
        if (past) pre = 8.2718061e-25f;  // 2^-80
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] *= pre;
        look(1);
    }
    // (2^-160 eps may be nothing: a row of one large value is then zeros and not 0 / 0)
    float v = var + a.eps * pre * pre;
    if (v < 1.1754944e-38f && pre != 1.f) v = 1.1754944e-38f;
    const float r = rsqrtf(v);
    if (me == 0 && cols) {
        if (a.mean) a.mean[row] = (mean + off) / pre;
        if (a.rstd) a.rstd[row] = r * pre;
    }
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) h[u][j] = ((h[u][j] - mean) - off) * r;
        if (a.weight) {
            float w[kVec];
            load8<TEAM, VEC, true>(a.weight, 0, a.weight_type, u, me, a.cols, w);
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] *= w[j];
        }
        if (a.bias) {
            float b[kVec];
            load8<TEAM, VEC, true>(a.bias, 0, a.weight_type, u, me, a.cols, b);
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] += b[j];
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            if (column<TEAM, VEC>(u, VEC ? 0 : j, me) < a.cols) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(h[u][j])));
    }
    if (a.scale_mode != kScaleNone) {
        float scale;
        if (a.scale_mode == kScaleRow) {
            // as bits a NaN is above every number
            const uint32_t most = team_max<TEAM>(__float_as_uint(top) & 0x7fffffffu, red.top);
            scale = __uint_as_float(max(most, __float_as_uint(1e-30f))) * (a.y_type == kTokI8 ? 1.f / 127.f : 1.f / 448.f);
            if (me == 0 && cols) a.scale[row] = scale;
        } else {
            scale = a.scale[0];
        }
        const float times = 1.f / scale;
        if (fabsf(times) < INFINITY) {
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
#pragma unroll
                for (int j = 0; j < kVec; ++j) h[u][j] *= times;
        } else {  // a scale near zero
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
#pragma unroll
                for (int j = 0; j < kVec; ++j) h[u][j] = __fdiv_rn(h[u][j], scale);
        }
    }
    if (a.y_type == kTokI8) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) store8_i8<TEAM, VEC>(a.y, row * a.y_stride, u, me, cols, h[u]);
    } else {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) store8<TEAM, VEC>(a.y, row * a.y_stride, a.y_type, u, me, cols, h[u]);
    }
}

// TEAM threads a row, TURNS times eight values each.
template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM == 32 ? 128 : TEAM) layer_norm_kernel(const __grid_constant__ LayerNormArgs a) {
    __shared__ Red red;
    const int me = threadIdx.x % TEAM;
    const int64_t row = TEAM == 32 ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (row >= a.rows) return;
    float h[TURNS][kVec];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) load8<TEAM, VEC, false>(a.x, row * a.x_stride, a.x_type, u, me, a.cols, h[u]);
    if (a.residual) {
        float r[TURNS][kVec];
#pragma unroll
        for (int u = 0; u < TURNS; ++u) load8<TEAM, VEC, false>(a.residual, row * a.residual_stride, a.residual_type, u, me, a.cols, r[u]);
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] += r[u][j];
    }
    if (a.sum) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) store8<TEAM, VEC>(a.sum, row * a.sum_stride, a.residual_type, u, me, a.cols, h[u]);
    }
    finish_row<TEAM, TURNS, VEC>(a, row, me, a.cols, h, red);
}

// Many rows of 16-bit x (and residual): the blocks stay and walk over the rows, a row's values on their way while the row
// before it is worked on, so that memory does not wait for the reductions.
template <int TEAM, int TURNS, bool RES>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM) layer_norm_stream_kernel(const __grid_constant__ LayerNormArgs a) {
    __shared__ Red red[2];
    const int me = threadIdx.x % TEAM, per = TEAM <= 32 ? 128 / TEAM : 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per;
    int64_t row = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / TEAM;
    uint4 x[TURNS], r[RES ? TURNS : 1];
    auto fetch = [&](int64_t at) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            const int c = column<TEAM, true>(u, 0, me);
            if (at >= a.rows || c >= a.cols) continue;
            x[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + at * a.x_stride + c);
            if (RES) r[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.residual) + at * a.residual_stride + c);
        }
    };
    fetch(row);
    int turn = 0;
    const int64_t first = TEAM < 32 ? row - threadIdx.x % 32 / TEAM : row;  // of the warp's teams: they end together
    for (int64_t lead = first; lead < a.rows; lead += step, row += step, turn ^= 1) {
        float h[TURNS][kVec];
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            unpack8(x[u], a.x_type, h[u]);
            if (RES) {
                float f[kVec];
                unpack8(r[u], a.residual_type, f);
#pragma unroll
                for (int j = 0; j < kVec; ++j) h[u][j] += f[j];
            }
            if (row >= a.rows || column<TEAM, true>(u, 0, me) >= a.cols) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) h[u][j] = 0.f;
            }
        }
        fetch(row + step);
        const int cols = TEAM < 32 && row >= a.rows ? 0 : a.cols;  // a team past the last row stores nothing
        if (a.sum) {
#pragma unroll
            for (int u = 0; u < TURNS; ++u) store8<TEAM, true>(a.sum, row * a.sum_stride, a.residual_type, u, me, cols, h[u]);
        }
        finish_row<TEAM, TURNS, true>(a, row, me, cols, h, red[turn]);  // a row's barriers lie between two uses of a half of red
    }
}

template <int TEAM, int TURNS>
cudaError_t launch(const LayerNormArgs& a, bool vec, cudaStream_t s) {
    const int threads = TEAM == 32 ? 128 : TEAM, per = threads / TEAM;
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + per - 1) / per);
    count_launch();
    if (vec)
        layer_norm_kernel<TEAM, TURNS, true><<<grid, threads, 0, s>>>(a);
    else
        layer_norm_kernel<TEAM, TURNS, false><<<grid, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <int TEAM, int TURNS, bool RES>
cudaError_t launch_stream(const LayerNormArgs& a, cudaStream_t s) {
    auto* kern = layer_norm_stream_kernel<TEAM, TURNS, RES>;
    constexpr int threads = TEAM <= 32 ? 128 : TEAM, per = threads / TEAM;
    static std::atomic<int> known;  // blocks that are resident at once on an SM; the same on every sm_100
    int resident = known.load(std::memory_order_relaxed);
    if (!resident) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kern, threads, 0);
        if (e != cudaSuccess) return e;
        known.store(resident, std::memory_order_relaxed);
    }
    const int64_t need = (static_cast<int64_t>(a.rows) + per - 1) / per, fit = static_cast<int64_t>(sm_count()) * resident;
    count_launch();
    kern<<<static_cast<unsigned>(need < fit ? need : fit), threads, 0, s>>>(a);
    return cudaGetLastError();
}
template <int TEAM, int TURNS>
cudaError_t launch_stream(const LayerNormArgs& a, cudaStream_t s) {
    return a.residual ? launch_stream<TEAM, TURNS, true>(a, s) : launch_stream<TEAM, TURNS, false>(a, s);
}

}  // namespace

cudaError_t launch_layer_norm(const LayerNormArgs& a, cudaStream_t s) {
    const bool vec = a.cols % kVec == 0 && rows_of_eights(a.x, a.x_stride, a.x_type) &&
                     rows_of_eights(a.residual, a.residual_stride, a.residual_type) &&
                     rows_of_eights(a.sum, a.sum_stride, a.residual_type) && rows_of_eights(a.weight, 0, a.weight_type) &&
                     rows_of_eights(a.bias, 0, a.weight_type) && rows_of_eights(a.y, a.y_stride, a.y_type);
    // the RMS norm's teams and its rule: little work takes a block a row, more of it blocks that stay
    const int64_t sms = sm_count();
    const bool few = a.cols <= 256 ? a.rows <= sms * 2 : static_cast<int64_t>(a.rows) * a.cols <= sms * 8192;
    if (vec && !few && a.x_type != kTokF32 && (!a.residual || a.residual_type != kTokF32)) {
        if (a.cols <= 64) return launch_stream<8, 1>(a, s);
        if (a.cols <= 128) return launch_stream<8, 2>(a, s);
        if (a.cols <= 256) return launch_stream<8, 4>(a, s);
        if (a.cols <= 320) return launch_stream<8, 5>(a, s);
        if (a.cols <= 512) return launch_stream<16, 4>(a, s);
        if (a.cols <= 1024) return launch_stream<32, 4>(a, s);
        if (a.cols <= 2048) return launch_stream<128, 2>(a, s);
        if (a.cols <= 4096) return launch_stream<256, 2>(a, s);
        if (a.cols <= 5120) return launch_stream<320, 2>(a, s);
        if (a.cols <= 6144) return launch_stream<384, 2>(a, s);
        if (a.cols <= 8192) return launch_stream<512, 2>(a, s);
        if (a.cols <= 16384) return launch_stream<1024, 2>(a, s);
    }
    if (a.cols <= 256) return launch<32, 1>(a, vec, s);
    if (a.cols <= 512) return launch<32, 2>(a, vec, s);
    if (a.cols <= 1024) return few ? launch<128, 1>(a, vec, s) : launch<32, 4>(a, vec, s);
    if (a.cols <= 2048) return launch<256, 1>(a, vec, s);
    if (a.cols <= 4096) return launch<512, 1>(a, vec, s);
    if (a.cols <= 5120) return launch<640, 1>(a, vec, s);
    if (a.cols <= 6144) return launch<768, 1>(a, vec, s);
    if (a.cols <= 7168) return launch<896, 1>(a, vec, s);
    if (a.cols <= 8192) return launch<1024, 1>(a, vec, s);
    if (a.cols <= 16384) return launch<1024, 2>(a, vec, s);
    return launch<1024, 4>(a, vec, s);
}

}  // namespace fxk
