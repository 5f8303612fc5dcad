// layer_norm_backward.cu — the layer norm's backward pass: the rows' gradient, and the sums over rows that are the
// gradients of weight and bias.
//
// With z = (h - mean) rstd and g = dy weight a row's gradient needs two sums, of g and of g z:
//   dx = (g - sum(g) / n - z sum(g z) / n) rstd + dsum,   dweight = sum over rows of dy z,   dbias = sum over rows of dy
// Bound by memory: dy, h, dsum and dx pass once. Blocks stay and walk over the rows; a thread holds the same columns of every
// row, so the sums over rows stay in its registers until its block's last row, and leave as one line of the workspace a
// block, which a second kernel adds up in a fixed order (4 us of the whole). Those sums take the registers of a third of the
// threads an SM could run, and what is left waits for its own results: 8192 x 4096 bf16 59 us, 4.5 TB/s, 69% of the copy;
// 100000 x 320 59 us; f32 8192 x 4096 120 us. Rows that are not aligned, a value at a time: 1031 x 5119 f16 26 us.
// Rows past 8192 columns would not leave room for the sums in registers: there the rows' gradient is a kernel of its own, and
// the sums over rows another, so dy and h pass twice (3004 x 9984 bf16 78 us).
#include "counters.hpp"
#include "token_rows.cuh"

#include <algorithm>
#include <atomic>

namespace fxk {
namespace {

constexpr int kFusedCols = 8192;
constexpr int kJoinedCols = 512;       // of rows that share a block
constexpr int kPlainSmem = 40 * 1024;  // dynamic shared memory that needs no asking for, beside a kernel's own

// A block's sums over its rows leave as its line of the workspace.
template <int TEAM, int TURNS, bool VEC>
__device__ __forceinline__ void leave_sums(const LayerNormBackwardArgs& a, int me, float (&dw)[TURNS][kVec], float (&db)[TURNS][kVec]) {
    constexpr int kThreads = TEAM <= 32 ? 128 : TEAM, kPer = kThreads / TEAM;
    extern __shared__ __align__(16) uint4 dynamic[];
    float* const joined = reinterpret_cast<float*>(dynamic);  // [2][cols]: the sums of a block of several teams
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
        __syncthreads();  // over the ring, which no team reads any more
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

// TEAM threads a row, TURNS times eight columns each.
template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM, TEAM == 256 || TEAM == 512 ? 1024 / TEAM : 1) layer_norm_backward_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    wait_for_earlier();
    constexpr int kThreads = TEAM <= 32 ? 128 : TEAM, kPer = kThreads / TEAM;
    __shared__ float2 red[2][32];
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
            if (a.weight) load8<TEAM, VEC, false>(a.weight, 0, a.weight_type, u, me, a.cols, w);
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
    leave_sums<TEAM, TURNS, VEC>(a, me, dw, db);
}

// Many rows of 16-bit values: the next rows' dy, h and dsum are on their way to shared memory while a row is worked on. TYPE: of
// dy, h, weight and dx alike, or -1: any. Where it says what the weights are, they are brought once a block and not once a row.
// Narrow rows take two values an instruction and hold the weights in shared memory, wide ones one value and registers, which
// leaves more of a row's work independent (bf16, us, the first and the second: 100000 x 320 59 and 75, 30000 x 1024 59 and 66,
// 8192 x 4096 62 and 59, 4000 x 8192 64 and 55).
constexpr int kAhead = 3;  // rows of a team in shared memory
template <int TEAM>
constexpr bool kNarrow = TEAM <= 128;
template <int TEAM, int TURNS>
constexpr int kRingBytes = (kAhead * 3 * (TEAM <= 32 ? 128 : TEAM) + (kNarrow<TEAM> ? TEAM : 0)) * TURNS * 16;  // and the weights

template <int TEAM, int TURNS, int TYPE>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM) layer_norm_backward_stream_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    wait_for_earlier();
    constexpr int kThreads = TEAM <= 32 ? 128 : TEAM, kPer = kThreads / TEAM;
    __shared__ float2 red[2][32];
    extern __shared__ __align__(16) uint4 dynamic[];
    uint4* const shared_held = dynamic;  // [turn][thread of a team]: narrow rows' weights
    uint4* const ring = dynamic + (kNarrow<TEAM> ? TURNS * TEAM : 0);  // [row][dy, h, dsum][turn][thread]
    const int me = threadIdx.x % TEAM;
    const float inv_n = 1.f / static_cast<float>(a.cols);
    float dw[TURNS][kVec] = {}, db[TURNS][kVec] = {};
    auto slot = [&](int at, int which, int u) { return ring + ((at * 3 + which) * TURNS + u) * kThreads + threadIdx.x; };
    auto fetch = [&](int64_t row, int at) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            const int c = column<TEAM, true>(u, 0, me);
            if (row >= a.rows || c >= a.cols) continue;
            copy16(slot(at, 0, u), static_cast<const uint16_t*>(a.dy) + row * a.dy_stride + c);
            copy16(slot(at, 1, u), static_cast<const uint16_t*>(a.h) + row * a.h_stride + c);
            if (a.dsum) copy16(slot(at, 2, u), static_cast<const uint16_t*>(a.dsum) + row * a.dsum_stride + c);
        }
        copies_end_row();
    };
    auto add = [](const float2& x, const float2& y) { return kNarrow<TEAM> ? add2(x, y) : make_float2(x.x + y.x, x.y + y.y); };
    auto mul = [](const float2& x, const float2& y) { return kNarrow<TEAM> ? mul2(x, y) : make_float2(x.x * y.x, x.y * y.y); };
    auto mul_add = [](const float2& x, const float2& y, const float2& z) {
        return kNarrow<TEAM> ? fma2(x, y, z) : make_float2(fmaf(x.x, y.x, z.x), fmaf(x.y, y.y, z.y));
    };
    uint4 held[TURNS];
    if (TYPE >= 0 && a.weight) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            const int c = column<TEAM, true>(u, 0, me);
            held[u] = c < a.cols ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.weight) + c) : make_uint4(0, 0, 0, 0);
            if (kNarrow<TEAM> && threadIdx.x < TEAM) shared_held[u * TEAM + me] = held[u];
        }
        if (kNarrow<TEAM>) __syncthreads();
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * kPer, mine = threadIdx.x / TEAM;
    int64_t lead = static_cast<int64_t>(blockIdx.x) * kPer;
    float mean = 0.f, rstd = 0.f;
    if (lead + mine < a.rows) mean = a.mean[lead + mine], rstd = a.rstd[lead + mine];
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i) fetch(lead + i * step + mine, i);
    for (int turn = 0, at = 0; lead < a.rows; lead += step, turn ^= 1) {
        const int64_t row = lead + mine;
        const int cols = row < a.rows ? a.cols : 0;  // lanes of no row run along: the sums are the warp's
        fetch(row + (kAhead - 1) * step, at == 0 ? kAhead - 1 : at - 1);
        copies_wait<kAhead - 1>();
        float g[TURNS][kVec], z[TURNS][kVec];
        const float2 m2 = make_float2(-mean, -mean), r2 = make_float2(rstd, rstd);
        if (row + step < a.rows) mean = a.mean[row + step], rstd = a.rstd[row + step];
        float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            if (column<TEAM, true>(u, 0, me) >= cols) continue;
            float w[kVec];
            unpack8(*slot(at, 0, u), TYPE < 0 ? a.dy_type : TYPE, g[u]);
            unpack8(*slot(at, 1, u), TYPE < 0 ? a.h_type : TYPE, z[u]);
            if (a.weight && TYPE >= 0)
                unpack8(kNarrow<TEAM> ? shared_held[u * TEAM + me] : held[u], TYPE, w);
            else if (a.weight)
                load8<TEAM, true, false>(a.weight, 0, a.weight_type, u, me, a.cols, w);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) {
                float2 gi = pair_of(g[u], i);
                const float2 zi = mul(add(pair_of(z[u], i), m2), r2);
                put_pair(dw[u], i, mul_add(gi, zi, pair_of(dw[u], i)));
                put_pair(db[u], i, add(pair_of(db[u], i), gi));
                if (a.weight) gi = mul(gi, pair_of(w, i));
                s1 = add(s1, gi);
                s2 = mul_add(gi, zi, s2);
                put_pair(g[u], i, gi);
                put_pair(z[u], i, zi);
            }
        }
        const float2 sums = team_sum2<TEAM>(make_float2(s1.x + s1.y, s2.x + s2.y), red[turn]);
        const float2 a1 = make_float2(-sums.x * inv_n, -sums.x * inv_n), a2 = make_float2(-sums.y * inv_n, -sums.y * inv_n);
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            if (column<TEAM, true>(u, 0, me) >= cols) continue;
            float more[kVec];
            if (a.dsum) unpack8(*slot(at, 2, u), TYPE < 0 ? a.dx_type : TYPE, more);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) {
                const float2 v = add(pair_of(g[u], i), mul_add(pair_of(z[u], i), a2, a1));
                put_pair(g[u], i, a.dsum ? mul_add(v, r2, pair_of(more, i)) : mul(v, r2));
            }
            store8<TEAM, true>(a.dx, row * a.dx_stride, TYPE < 0 ? a.dx_type : TYPE, u, me, cols, g[u]);
        }
        if (++at == kAhead) at = 0;
    }
    leave_sums<TEAM, TURNS, true>(a, me, dw, db);
}

// A block a row, of any length: its values are read twice.
constexpr int kWideThreads = 512;
template <bool VEC>
__global__ void __launch_bounds__(kWideThreads) layer_norm_backward_wide_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    wait_for_earlier();
    __shared__ float2 red[32];
    const int64_t row = blockIdx.x;
    const int me = threadIdx.x, turns = (a.cols + kWideThreads * kVec - 1) / (kWideThreads * kVec);
    const float mean = a.mean[row], rstd = a.rstd[row], inv_n = 1.f / static_cast<float>(a.cols);
    auto at = [&](int u, float (&g)[kVec], float (&z)[kVec]) {  // columns past the row are 0 in g
        load8<kWideThreads, VEC, false>(a.dy, row * a.dy_stride, a.dy_type, u, me, a.cols, g);
        load8<kWideThreads, VEC, false>(a.h, row * a.h_stride, a.h_type, u, me, a.cols, z);
        if (a.weight) {
            float w[kVec];
            load8<kWideThreads, VEC, false>(a.weight, 0, a.weight_type, u, me, a.cols, w);
#pragma unroll
            for (int j = 0; j < kVec; ++j) g[j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) z[j] = (z[j] - mean) * rstd;
    };
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int u = 0; u < turns; ++u) {
        float g[kVec], z[kVec];
        at(u, g, z);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            const bool inside = column<kWideThreads, VEC>(u, VEC ? 0 : j, me) < a.cols;
            sums.x += g[j];
            if (inside) sums.y = fmaf(g[j], z[j], sums.y);
        }
    }
    sums = team_sum2<kWideThreads>(sums, red);
    sums.x *= inv_n;
    sums.y *= inv_n;
#pragma unroll 2
    for (int u = 0; u < turns; ++u) {
        float g[kVec], z[kVec];
        at(u, g, z);
#pragma unroll
        for (int j = 0; j < kVec; ++j) g[j] = (g[j] - fmaf(z[j], sums.y, sums.x)) * rstd;
        if (a.dsum) {
            load8<kWideThreads, VEC, false>(a.dsum, row * a.dsum_stride, a.dx_type, u, me, a.cols, z);
#pragma unroll
            for (int j = 0; j < kVec; ++j) g[j] += z[j];
        }
        store8<kWideThreads, VEC>(a.dx, row * a.dx_stride, a.dx_type, u, me, a.cols, g);
    }
}

// The same of 16-bit rows up to 16384 columns, as they lie in memory in registers between the two looks at them.
constexpr int kHeldTurns = 4;
__global__ void __launch_bounds__(kWideThreads, 2) layer_norm_backward_held_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    wait_for_earlier();
    __shared__ float2 red[32];
    const int64_t row = blockIdx.x;
    const int me = threadIdx.x;
    uint4 dy[kHeldTurns], h[kHeldTurns];
#pragma unroll
    for (int u = 0; u < kHeldTurns; ++u) {
        const int c = column<kWideThreads, true>(u, 0, me);
        if (c >= a.cols) continue;
        dy[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.dy) + row * a.dy_stride + c);
        h[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.h) + row * a.h_stride + c);
    }
    const float mean = a.mean[row], rstd = a.rstd[row], inv_n = 1.f / static_cast<float>(a.cols);
    float2 sums = make_float2(0.f, 0.f);
    auto each = [&](auto&& then) {
#pragma unroll
        for (int u = 0; u < kHeldTurns; ++u) {
            if (column<kWideThreads, true>(u, 0, me) >= a.cols) continue;
            float g[kVec], z[kVec];
            unpack8(dy[u], a.dy_type, g);
            unpack8(h[u], a.h_type, z);
            if (a.weight) {
                float w[kVec];
                load8<kWideThreads, true, false>(a.weight, 0, a.weight_type, u, me, a.cols, w);
#pragma unroll
                for (int j = 0; j < kVec; ++j) g[j] *= w[j];
            }
#pragma unroll
            for (int j = 0; j < kVec; ++j) z[j] = (z[j] - mean) * rstd;
            then(u, g, z);
        }
    };
    each([&](int, float (&g)[kVec], float (&z)[kVec]) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            sums.x += g[j];
            sums.y = fmaf(g[j], z[j], sums.y);
        }
    });
    sums = team_sum2<kWideThreads>(sums, red);
    sums.x *= inv_n;
    sums.y *= inv_n;
    each([&](int u, float (&g)[kVec], float (&z)[kVec]) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) g[j] = (g[j] - fmaf(z[j], sums.y, sums.x)) * rstd;
        if (a.dsum) {
            load8<kWideThreads, true, false>(a.dsum, row * a.dsum_stride, a.dx_type, u, me, a.cols, z);
#pragma unroll
            for (int j = 0; j < kVec; ++j) g[j] += z[j];
        }
        store8<kWideThreads, true>(a.dx, row * a.dx_stride, a.dx_type, u, me, a.cols, g);
    });
}

// Sums over rows alone: a block takes 256 columns and every gridDim.y-th row.
__global__ void __launch_bounds__(256) layer_norm_sums_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    wait_for_earlier();
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

// The same of rows aligned to eights: a warp takes 256 columns and every eighth of the block's rows. ALL16: of 16-bit values,
// four rows on their way at a time.
template <bool ALL16>
__global__ void __launch_bounds__(256) layer_norm_sums8_kernel(const __grid_constant__ LayerNormBackwardArgs a) {
    wait_for_earlier();
    constexpr int kRows = 4;
    __shared__ float part[8][32 * kVec + 4];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c0 = blockIdx.x * (32 * kVec);
    const int cols = min(32 * kVec, a.cols - c0);
    float dw[kVec] = {}, db[kVec] = {};
    const int64_t step = static_cast<int64_t>(gridDim.y) * 8;
    auto take = [&](float (&g)[kVec], float (&z)[kVec], float mean, float rstd) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            dw[j] = fmaf(g[j], (z[j] - mean) * rstd, dw[j]);
            db[j] += g[j];
        }
    };
    for (int64_t row0 = static_cast<int64_t>(blockIdx.y) * 8 + warp; row0 < a.rows; row0 += kRows * step) {
        if (ALL16) {
            uint4 dy[kRows], h[kRows];
            float mean[kRows], rstd[kRows];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int64_t row = row0 + i * step;
                if (row >= a.rows || lane * kVec >= cols) break;
                dy[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.dy) + row * a.dy_stride + c0 + lane * kVec);
                h[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.h) + row * a.h_stride + c0 + lane * kVec);
                mean[i] = a.mean[row], rstd[i] = a.rstd[row];
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                if (row0 + i * step >= a.rows || lane * kVec >= cols) break;
                float g[kVec], z[kVec];
                unpack8(dy[i], a.dy_type, g);
                unpack8(h[i], a.h_type, z);
                take(g, z, mean[i], rstd[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int64_t row = row0 + i * step;
                if (row >= a.rows) break;
                float g[kVec], z[kVec];
                load8<32, true, false>(a.dy, row * a.dy_stride + c0, a.dy_type, 0, lane, cols, g);
                load8<32, true, false>(a.h, row * a.h_stride + c0, a.h_type, 0, lane, cols, z);
                take(g, z, a.mean[row], a.rstd[row]);
            }
        }
    }
    float* const mine = a.work + static_cast<int64_t>(blockIdx.y) * 2 * a.cols + c0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kVec; ++j) part[warp][lane * kVec + j] = which ? db[j] : dw[j];
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < cols) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) sum += part[w][threadIdx.x];
            mine[which * a.cols + threadIdx.x] = sum;
        }
    }
}

// The lines of the workspace added up: 32 columns a block, eight warps that take every eighth line.
__global__ void __launch_bounds__(256) layer_norm_join_kernel(const float* work, int lines, int cols, float* dweight, float* dbias,
                                                             bool accumulate) {
    __shared__ float part[8][33];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;  // of dweight and dbias in a row
    const int warp = threadIdx.x / 32;
    float s = 0.f;
    wait_for_earlier();
    if (c < 2 * cols)
#pragma unroll 8
        for (int i = warp; i < lines; i += 8) s += __ldcg(work + static_cast<int64_t>(i) * 2 * cols + c);  // written while this kernel began
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

template <int TEAM, class Kernel>
cudaError_t launch(const LayerNormBackwardArgs& a, Kernel* kern, int ring, std::atomic<int>& known, int& lines, cudaStream_t s) {
    constexpr int threads = TEAM <= 32 ? 128 : TEAM, per = threads / TEAM;
    const int bytes = std::max(per > 1 ? 8 * kJoinedCols : 0, ring);
    if (bytes > kPlainSmem) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
    }
    int resident = known.load(std::memory_order_relaxed);
    if (!resident) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kern, threads, bytes);
        if (e != cudaSuccess) return e;
        known.store(resident, std::memory_order_relaxed);
    }
    const int64_t need = (static_cast<int64_t>(a.rows) + per - 1) / per, fit = static_cast<int64_t>(sm_count()) * resident;
    lines = static_cast<int>(std::min({need, fit, layer_norm_backward_blocks(a.rows, a.cols)}));
    count_launch();
    return launch_early(kern, dim3(static_cast<unsigned>(lines)), threads, bytes, s, a);
}
template <int TEAM, int TURNS>
cudaError_t launch(const LayerNormBackwardArgs& a, bool vec, int& lines, cudaStream_t s) {
    static std::atomic<int> known[2];  // blocks that are resident at once on an SM; the same on every sm_100
    return vec ? launch<TEAM>(a, layer_norm_backward_kernel<TEAM, TURNS, true>, 0, known[1], lines, s)
               : launch<TEAM>(a, layer_norm_backward_kernel<TEAM, TURNS, false>, 0, known[0], lines, s);
}
template <int TEAM, int TURNS>
cudaError_t launch_stream(const LayerNormBackwardArgs& a, int& lines, cudaStream_t s) {
    static std::atomic<int> known[3];
    constexpr int ring = kRingBytes<TEAM, TURNS>;
    const int t = a.dy_type;
    if (a.h_type != t || a.dx_type != t || (a.weight && a.weight_type != t))
        return launch<TEAM>(a, layer_norm_backward_stream_kernel<TEAM, TURNS, -1>, ring, known[0], lines, s);
    return t == kTokF16 ? launch<TEAM>(a, layer_norm_backward_stream_kernel<TEAM, TURNS, kTokF16>, ring, known[1], lines, s)
                        : launch<TEAM>(a, layer_norm_backward_stream_kernel<TEAM, TURNS, kTokBF16>, ring, known[2], lines, s);
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
    const bool vec_in = a.cols % kVec == 0 && rows_of_eights(a.dy, a.dy_stride, a.dy_type) && rows_of_eights(a.h, a.h_stride, a.h_type);
    const bool vec = vec_in && rows_of_eights(a.weight, 0, a.weight_type) && rows_of_eights(a.dsum, a.dsum_stride, a.dx_type) &&
                     rows_of_eights(a.dx, a.dx_stride, a.dx_type);
    const bool stream = vec && a.dy_type != kTokF32 && a.h_type != kTokF32 && (!a.dsum || a.dx_type != kTokF32);
    if (a.cols > kFusedCols || !a.dx) {
        if (a.work) {
            // enough blocks to fill the GPU several times (3004 x 9984 bf16: 182 us in all with a value a thread in both kernels)
            const int64_t across = (a.cols + 255) / 256, most = layer_norm_backward_blocks(a.rows, a.cols);
            lines = static_cast<int>(std::min({most, (static_cast<int64_t>(a.rows) + 7) / 8,
                                               vec_in ? std::max<int64_t>(8 * sm_count() / across, 1) : most}));
            count_launch();
            auto* kern = !vec_in                                              ? layer_norm_sums_kernel
                         : a.dy_type != kTokF32 && a.h_type != kTokF32 ? layer_norm_sums8_kernel<true>
                                                                       : layer_norm_sums8_kernel<false>;
            e = launch_early(kern, dim3(static_cast<unsigned>(across), lines), 256, 0, s, a);
        }
        if (a.dx && e == cudaSuccess) {  // after the sums: dx may take its place over dy or h
            const bool held = vec && a.cols <= kHeldTurns * kWideThreads * kVec && a.dy_type != kTokF32 && a.h_type != kTokF32;
            auto* kern = held ? layer_norm_backward_held_kernel
                         : vec ? layer_norm_backward_wide_kernel<true>
                               : layer_norm_backward_wide_kernel<false>;
            count_launch();
            e = launch_early(kern, dim3(a.rows), kWideThreads, 0, s, a);
        }
    } else {
        if (stream)
            e = a.cols <= 64     ? launch_stream<8, 1>(a, lines, s)
                : a.cols <= 128  ? launch_stream<16, 1>(a, lines, s)
                : a.cols <= 256  ? launch_stream<32, 1>(a, lines, s)
                : a.cols <= 512  ? launch_stream<32, 2>(a, lines, s)
                : a.cols <= 1024 ? launch_stream<128, 1>(a, lines, s)
                : a.cols <= 2048 ? launch_stream<128, 2>(a, lines, s)
                : a.cols <= 4096 ? launch_stream<256, 2>(a, lines, s)
                : a.cols <= 5120 ? launch_stream<320, 2>(a, lines, s)
                : a.cols <= 6144 ? launch_stream<384, 2>(a, lines, s)
                                 : launch_stream<512, 2>(a, lines, s);
        else if (a.cols <= 64)
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
    return launch_early(layer_norm_join_kernel, dim3((2 * a.cols + 31) / 32), 256, 0, s, a.work, lines, a.cols, a.dweight, a.dbias,
                        a.accumulate);
}

}  // namespace fxk
