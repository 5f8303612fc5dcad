// rms_norm.cu — root-mean-square norm of token rows with the residual's addition and 8-bit output.
//
// Bound by memory: x, residual, sum and y pass once (7 bytes a value for bf16 to e4m3). A row's h = x + residual
// stays in the registers of its team of threads, eight consecutive values a thread and turn, between the three
// looks at it: the sum of squares, the largest magnitude, the output. A team is a part of a warp, a warp or a block.
// Where rows are many, blocks stay and walk over them with the next row's loads on their way during a row's
// reductions (16384 x 4096 bf16 with residual to e4m3: 75 us, 6.2 TB/s; 99 us with a block a row); where they are few,
// a block a row has as many threads as the row has eights (1 x 4096: 2.5 us, launch and two reductions). Rows that are
// no multiple of eight values, or not aligned, are read one value at a time, neighbours by neighbours (1031 x 5119 f16
// with residual: 15.5 us, 2.4 TB/s, bound by a load and a store a value, this form's own; with the next row brought to
// shared memory in 16-byte pieces 19).
#include "counters.hpp"
#include "token_rows.cuh"

#include <atomic>

namespace fxk {
namespace {

// From a row's h on: the norm, the scale, the output; cols 0: no row, nothing is stored. red: three rows of 32 floats that
// no thread of the team still reads.
template <int TEAM, int TURNS, bool VEC>
__device__ __forceinline__ void finish_row(const RmsNormArgs& a, int64_t row, int me, int cols, float (&h)[TURNS][kVec],
                                           float (*red)[32]) {
    float ss = 0.f;
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
#pragma unroll
        for (int j = 0; j < kVec; ++j) ss = fmaf(h[u][j], h[u][j], ss);
    ss = team_sum<TEAM>(ss, red[0]);
    float pre = 1.f;
    // squares (and eps) past f32's range, or a NaN or infinity, which stays one: sum smaller ones
    const bool past = !(ss + a.eps < 3.0e38f);
    if (TEAM < 32 ? __any_sync(0xffffffffu, past) : past) {
        if (past) pre = 8.2718061e-25f;  // 2^-80
        ss = 0.f;
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                h[u][j] *= pre;
                ss = fmaf(h[u][j], h[u][j], ss);
            }
        ss = team_sum<TEAM>(ss, red[1]);
    }
    const float r = rsqrtf(ss / static_cast<float>(a.cols) + a.eps * pre * pre);
    // v = h weight r: r joins the scale, so that a value takes two products
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        if (a.weight) {
            float w[kVec];
            load8<TEAM, VEC, true>(a.weight, 0, a.weight_type, u, me, a.cols, w);
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j)  // columns past the row are 0
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(h[u][j])));
    }
    float times = r, scale = 1.f;
    if (a.scale_mode == kScaleRow) {
        // as bits a NaN is above every number
        const uint32_t most = team_max<TEAM>(__float_as_uint(top * r) & 0x7fffffffu, reinterpret_cast<uint32_t*>(red[2]));
        scale = __uint_as_float(max(most, __float_as_uint(1e-30f))) * (1.f / 448.f);
        if (me == 0 && cols) a.scale[row] = scale;
        times = r * (1.f / scale);
    } else if (a.scale_mode == kScaleTensor) {
        scale = a.scale[0];
        times = r * (1.f / scale);
    }
    // a row near zero under a small eps, or a scale near zero: one product after the other (zeros stay zeros)
    if (fabsf(times) == INFINITY) {
        const float inv = 1.f / (scale * 1.8446744e19f);  // 2^64
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] = h[u][j] * r * inv;
        times = 1.8446744e19f;
    }
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) h[u][j] *= times;
        store8<TEAM, VEC>(a.y, row * a.y_stride, a.y_type, u, me, cols, h[u]);
    }
}

// TEAM threads a row, TURNS times eight values each.
template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM == 32 ? 128 : TEAM) rms_norm_kernel(const __grid_constant__ RmsNormArgs a) {
    __shared__ float red[3][32];
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
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM) rms_norm_stream_kernel(const __grid_constant__ RmsNormArgs a) {
    __shared__ float red[2][3][32];
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
            if (column<TEAM, true>(u, 0, me) >= a.cols) {
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
        finish_row<TEAM, TURNS, true>(a, row, me, cols, h, red[turn]);  // a row's barrier lies between two uses of a half of red
    }
}

template <int TEAM, int TURNS>
cudaError_t launch(const RmsNormArgs& a, bool vec, cudaStream_t s) {
    const int threads = TEAM == 32 ? 128 : TEAM, per = threads / TEAM;
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + per - 1) / per);
    count_launch();
    if (vec)
        rms_norm_kernel<TEAM, TURNS, true><<<grid, threads, 0, s>>>(a);
    else
        rms_norm_kernel<TEAM, TURNS, false><<<grid, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <int TEAM, int TURNS, bool RES>
cudaError_t launch_stream(const RmsNormArgs& a, cudaStream_t s) {
    auto* kern = rms_norm_stream_kernel<TEAM, TURNS, RES>;
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
cudaError_t launch_stream(const RmsNormArgs& a, cudaStream_t s) {
    return a.residual ? launch_stream<TEAM, TURNS, true>(a, s) : launch_stream<TEAM, TURNS, false>(a, s);
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormArgs& a, cudaStream_t s) {
    auto ok = [&](const void* p, int64_t stride, int type) {  // 16-byte aligned rows (8-byte of e4m3)
        const int64_t size = type == kTokF32 ? 4 : type == kTokE4M3 ? 1 : 2, unit = type == kTokE4M3 ? 8 : 16;
        return !p || (reinterpret_cast<uintptr_t>(p) % unit == 0 && stride * size % unit == 0);
    };
    const bool vec = a.cols % kVec == 0 && ok(a.x, a.x_stride, a.x_type) && ok(a.residual, a.residual_stride, a.residual_type) &&
                     ok(a.sum, a.sum_stride, a.residual_type) && ok(a.weight, 0, a.weight_type) && ok(a.y, a.y_stride, a.y_type);
    // little work: a block a row with as many threads as it has eights, for the shortest way through; more: blocks that stay
    // (us, the one and the other: 444 x 320 3.2 and 4.0, 4736 x 320 6.1 and 6.2, 9472 x 320 10.3 and 7.1, 222 x 4096 4.3
    // and 4.4, 370 x 8192 8.8 and 7.5; rows of eights to a warp's quarter: 444 x 64 2.3 and 1.8)
    const int64_t sms = sm_count();
    const bool few = a.cols <= 256 ? a.rows <= sms * 2 : static_cast<int64_t>(a.rows) * a.cols <= sms * 8192;
    if (vec && !few && a.x_type != kTokF32 && (!a.residual || a.residual_type != kTokF32)) {
        // narrow rows: several to a warp, so that its lanes are busy and have loads enough on their way (200003 x 320 bf16
        // to bf16: 50 us, 69 with a warp a row)
        if (a.cols <= 64) return launch_stream<8, 1>(a, s);
        if (a.cols <= 128) return launch_stream<8, 2>(a, s);
        if (a.cols <= 256) return launch_stream<8, 4>(a, s);
        if (a.cols <= 320) return launch_stream<8, 5>(a, s);
        if (a.cols <= 512) return launch_stream<16, 4>(a, s);
        if (a.cols <= 1024) return launch_stream<32, 4>(a, s);
        if (a.cols <= 2048) return launch_stream<128, 2>(a, s);
        if (a.cols <= 4096) return launch_stream<256, 2>(a, s);
        // (8192 x 5120 51 us, 64 with 512 threads; a team of 448 for 7168 columns is no faster)
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
    // (teams between the powers of two: 1031 x 5119 15 us, 20 with 1024 threads)
    if (a.cols <= 5120) return launch<640, 1>(a, vec, s);
    if (a.cols <= 6144) return launch<768, 1>(a, vec, s);
    if (a.cols <= 7168) return launch<896, 1>(a, vec, s);
    if (a.cols <= 8192) return launch<1024, 1>(a, vec, s);
    if (a.cols <= 16384) return launch<1024, 2>(a, vec, s);
    return launch<1024, 4>(a, vec, s);
}

}  // namespace fxk
