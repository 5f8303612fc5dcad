// layer_norm.cu — layer norm of token rows with the residual's addition, the rows' statistics and 8-bit output.
//
// Bound by memory, as the RMS norm: x, residual, sum and y pass once, a row stays in the registers of its team of threads
// between the looks at it (its mean, its squares about it, its largest magnitude where it gets a scale, its output), blocks
// stay and walk over many rows with the next row on its way. What a value then costs are instructions: pairs of values share
// one (add, multiply, multiply-add of two f32), and a kernel has one type (16384 x 4096 bf16 with residual to bf16 85 us, 6.3
// TB/s, 96% of the copy, 107 before that; to e4m3 or i8 96 us; without a residual 63 us, 4.2 TB/s, bound by a row's three
// reductions' way through a block; 1 x 4096 3.0 us). Rows that are not aligned, read a value at a time: 1031 x 5119 22 us.
// The variance is the mean square about the mean, not a difference of two sums, so that rows far from zero keep theirs:
// t = h - mean is exact or rounded once, and the sum of the t, taken with that of their squares, gives what the mean
// itself was off by. Where that is more than the values are spread, both sums are taken again.
#include "counters.hpp"
#include "token_rows.cuh"

#include <atomic>

namespace fxk {
namespace {

constexpr float kSmaller = 8.2718061e-25f;  // 2^-80
constexpr int kAgain = 13;  // times that squares are summed again, at most: each takes 17 bits or more (80 roundings) off what the mean is off by

struct Red {  // of a block that is one team: a row's sums, one of each look
    float2 pair[2][32];
    float sum[2][32];
    uint32_t top[32];
};

// Scale of a row from its largest magnitude: a quotient by 127 or 448, correctly rounded (the product with the reciprocal, made good by its
// remainder: of every f32 from 1e-30 on). Infinity and NaN stay.
__device__ __forceinline__ float row_scale(float top, int y_type) {
    const float by = y_type == kTokI8 ? 127.f : 448.f, inv = y_type == kTokI8 ? 1.f / 127.f : 1.f / 448.f, t = top * inv;
    return t < INFINITY ? fmaf(fmaf(t, -by, top), inv, t) : t;
}

// From a row's h on; cols 0: no row, nothing is stored. red: no thread of the team still reads it.
// TYPE: of x, residual, weight and bias alike, or -1: any.
template <int TEAM, int TURNS, bool VEC, int TYPE>
__device__ __forceinline__ void finish_row(const LayerNormArgs& a, int64_t row, int me, int cols, float (&h)[TURNS][kVec],
                                           Red& red) {
    const float inv_n = 1.f / static_cast<float>(a.cols);
    auto inside = [&](int u, int j) { return column<TEAM, VEC>(u, j, me) < a.cols; };  // with VEC of all eight alike
    auto scaled = [&](float by) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[u][j] *= by;
    };
    auto total = [&](float* to) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) s = add2(s, pair_of(h[u], i));  // columns past the row are 0
        return team_sum1<TEAM>(s.x + s.y, to);
    };
    float pre = 1.f;
    float s = total(red.sum[0]);
    // a sum past f32's range, or a NaN or infinity, which stays one: sum smaller values
    const bool past = !(fabsf(s) < 3.0e38f);
    if (TEAM < 32 ? __any_sync(0xffffffffu, past) : past) {
        if (past) pre = kSmaller;
        scaled(pre);
        s = total(red.sum[1]);
    }
    float mean = s * inv_n;  // what this and the sum are off by, off has
    // t = h - mean in h's place; their sum and that of their squares
    auto squares = [&](float less, float2* to) {
        float2 e = make_float2(0.f, 0.f), q = e;
        const float2 m = make_float2(-less, -less);
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            if (VEC && !inside(u, 0)) continue;
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) {
                float2 t = add2(pair_of(h[u], i), m);
                if (!VEC) t = make_float2(inside(u, 2 * i) ? t.x : 0.f, inside(u, 2 * i + 1) ? t.y : 0.f);
                put_pair(h[u], i, t);
                e = add2(e, t);
                q = fma2(t, t, q);
            }
        }
        return team_sum2<TEAM>(make_float2(e.x + e.y, q.x + q.y), to);
    };
    float2 q = squares(mean, red.pair[0]);
    float off = q.x * inv_n, var = fmaxf(q.y * inv_n - off * off, 0.f) + a.eps * pre * pre;
    // Squares past f32's range; or a mean further off than the values are spread (rows nearly or all alike, far from zero), which leaves of
    // the squares mostly their rounding: they are summed again, of smaller values, or about the better mean.
    const bool again = !(off * off <= var && q.y + a.eps < 3.0e38f);
    if (__builtin_expect(TEAM < 32 ? __any_sync(0xffffffffu, again) : again, 0)) {
        for (int i = 0; i < kAgain; ++i) {
            const bool wide = !(q.y + a.eps < 3.0e38f) && pre == 1.f, far = !wide && off * off > var;
            if (!(TEAM < 32 ? __any_sync(0xffffffffu, wide || far) : wide || far)) break;
            const float by = wide ? kSmaller : 1.f, less = far ? off : 0.f;
            pre *= by;
            mean = mean * by + less;
            scaled(by);
            q = squares(less, red.pair[(i + 1) % 2]);  // not the half that slower threads may still read
            off = q.x * inv_n;
            var = fmaxf(q.y * inv_n - off * off, 0.f) + a.eps * pre * pre;
        }
    }
    float undo = pre;
    // 2^-160 eps may be nothing: what is left then are values all alike
    if (var < 1.1754944e-38f && pre != 1.f) var = a.eps, undo = 1.f;
    if (!(q.y < INFINITY)) var = q.y - q.y;  // a value or a difference that is not finite: NaN
    const float r = rsqrtf(var);
    if (me == 0 && cols) {
        if (a.mean) a.mean[row] = (mean + off) / pre;
        if (a.rstd) a.rstd[row] = r * undo;
    }
    const float2 r2 = make_float2(r, r), off2 = make_float2(-off * r, -off * r);
    const bool by_row = a.scale_mode == kScaleRow;
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        if (VEC && !inside(u, 0)) continue;
        float w[kVec], b[kVec];
        if (a.weight) load8<TEAM, VEC, false>(a.weight, 0, TYPE < 0 ? a.weight_type : TYPE, u, me, a.cols, w);
        if (a.bias) load8<TEAM, VEC, false>(a.bias, 0, TYPE < 0 ? a.weight_type : TYPE, u, me, a.cols, b);
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
            float2 v = fma2(pair_of(h[u], i), r2, off2);
            if (a.weight && a.bias)
                v = fma2(v, pair_of(w, i), pair_of(b, i));
            else if (a.weight)
                v = mul2(v, pair_of(w, i));
            else if (a.bias)
                v = add2(v, pair_of(b, i));
            put_pair(h[u], i, v);
        }
        if (by_row) {
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) {
                const float2 v = pair_of(h[u], i);
                top = max_abs(top, VEC ? v : make_float2(inside(u, 2 * i) ? v.x : 0.f, inside(u, 2 * i + 1) ? v.y : 0.f));
            }
        }
    }
    float scale = 1.f;
    if (a.scale_mode != kScaleNone) {
        bool zeros = false;
        if (by_row) {
            const uint32_t most = team_max<TEAM>(__float_as_uint(top), red.top);  // as bits a NaN is above every number
            zeros = most == 0;
            scale = row_scale(__uint_as_float(max(most, __float_as_uint(1e-30f))), a.y_type);
            if (me == 0 && cols) a.scale[row] = scale;
        } else {
            scale = a.scale[0];
        }
        // v / scale rounded to f32, as the quantiser has it, so that a row's codes are those of its f32 values (16384 x 4096 bf16 to
        // e4m3 or i8 94 us, 88 by a product with the reciprocal alone). Below 1e-20 and from 1e37 on terms of quotient2 could leave
        // f32's normal numbers, but for rows of zeros.
        const bool within = (fabsf(scale) > 1e-20f && fabsf(scale) < 1e37f) || zeros;
        const float inv = 1.f / scale;
        const float2 inv2 = make_float2(inv, inv), less2 = make_float2(-scale, -scale);
        auto divided = [&](auto&& by) {
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
#pragma unroll
                for (int i = 0; i < kVec / 2; ++i) put_pair(h[u], i, by(pair_of(h[u], i)));
        };
        if (within && by_row) {  // no quotient is past 448
            divided([&](const float2& v) { return quotient2(v, inv2, less2); });
        } else if (within) {  // those far above saturate as they are
            divided([&](const float2& v) {
                const float2 t = mul2(v, inv2), q = quotient2(v, inv2, less2);
                return make_float2(fabsf(t.x) < 512.f ? q.x : t.x, fabsf(t.y) < 512.f ? q.y : t.y);
            });
        } else {
            divided([&](const float2& v) { return make_float2(__fdiv_rn(v.x, scale), __fdiv_rn(v.y, scale)); });
        }
    }
    // (a row's own scale leaves no value above 127)
    const bool plain = by_row && scale < INFINITY;
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        if (a.y_type != kTokI8)
            store8<TEAM, VEC>(a.y, row * a.y_stride, a.y_type, u, me, cols, h[u]);
        else if (VEC && plain)
            store8_i8_within<TEAM>(a.y, row * a.y_stride, u, me, cols, h[u]);
        else
            store8_i8<TEAM, VEC>(a.y, row * a.y_stride, u, me, cols, h[u]);
    }
}

// TEAM threads a row, TURNS times eight values each.
template <int TEAM, int TURNS, bool VEC>
__global__ void __launch_bounds__(TEAM == 32 ? 128 : TEAM) layer_norm_kernel(const __grid_constant__ LayerNormArgs a) {
    wait_for_earlier();
    let_later_begin();
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
    finish_row<TEAM, TURNS, VEC, -1>(a, row, me, a.cols, h, red);
}

// Many rows of 16-bit x (and residual): the blocks stay and walk over the rows, a row's values on their way while the row
// before it is worked on, so that memory does not wait for the reductions.
template <int TEAM, int TURNS, bool RES, int TYPE>
__global__ void __launch_bounds__(TEAM <= 32 ? 128 : TEAM) layer_norm_stream_kernel(const __grid_constant__ LayerNormArgs a) {
    wait_for_earlier();
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
            unpack8(x[u], TYPE < 0 ? a.x_type : TYPE, h[u]);
            if (RES) {
                float f[kVec];
                unpack8(r[u], TYPE < 0 ? a.residual_type : TYPE, f);
#pragma unroll
                for (int i = 0; i < kVec / 2; ++i) put_pair(h[u], i, add2(pair_of(h[u], i), pair_of(f, i)));
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
        finish_row<TEAM, TURNS, true, TYPE>(a, row, me, cols, h, red[turn]);  // a row's barriers lie between two uses of a half of red
    }
}

// The same with the next rows' values on their way to shared memory: rows so long that a block's registers would hold the
// values on their way of no second block (8192 x 8192 bf16 with residual 97 us, 110 with them in registers; but 16384 x 4096 91
// for 85, 16384 x 1024 31 for 27: a copy and a read more a value).
constexpr int kAhead = 3;  // rows in shared memory
template <int TEAM, int TURNS, bool RES>
constexpr int kRingBytes = kAhead * (RES ? 2 : 1) * TURNS * TEAM * 16;

template <int TEAM, int TURNS, bool RES, int TYPE>
__global__ void __launch_bounds__(TEAM) layer_norm_ring_kernel(const __grid_constant__ LayerNormArgs a) {
    wait_for_earlier();
    __shared__ Red red[2];
    extern __shared__ __align__(16) uint4 ring[];  // [row][x, residual][turn][thread]
    const int me = threadIdx.x;
    const int64_t step = gridDim.x;
    auto slot = [&](int at, int which, int u) { return ring + ((at * (RES ? 2 : 1) + which) * TURNS + u) * TEAM + me; };
    auto fetch = [&](int64_t row, int at) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            const int c = column<TEAM, true>(u, 0, me);
            if (row >= a.rows || c >= a.cols) continue;
            copy16(slot(at, 0, u), static_cast<const uint16_t*>(a.x) + row * a.x_stride + c);
            if (RES) copy16(slot(at, 1, u), static_cast<const uint16_t*>(a.residual) + row * a.residual_stride + c);
        }
        copies_end_row();
    };
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i) fetch(blockIdx.x + i * step, i);
    int64_t row = blockIdx.x;
    for (int turn = 0, at = 0; row < a.rows; row += step, turn ^= 1) {
        fetch(row + (kAhead - 1) * step, at == 0 ? kAhead - 1 : at - 1);
        copies_wait<kAhead - 1>();
        float h[TURNS][kVec];
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            if (column<TEAM, true>(u, 0, me) >= a.cols) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) h[u][j] = 0.f;
                continue;
            }
            unpack8(*slot(at, 0, u), TYPE < 0 ? a.x_type : TYPE, h[u]);
            if (RES) {
                float f[kVec];
                unpack8(*slot(at, 1, u), TYPE < 0 ? a.residual_type : TYPE, f);
#pragma unroll
                for (int i = 0; i < kVec / 2; ++i) put_pair(h[u], i, add2(pair_of(h[u], i), pair_of(f, i)));
            }
            if (a.sum) store8<TEAM, true>(a.sum, row * a.sum_stride, a.residual_type, u, me, a.cols, h[u]);
        }
        if (++at == kAhead) at = 0;
        finish_row<TEAM, TURNS, true, TYPE>(a, row, me, a.cols, h, red[turn]);  // a row's barriers lie between two uses of a half of red
    }
}

template <int TEAM, int TURNS>
cudaError_t launch(const LayerNormArgs& a, bool vec, cudaStream_t s) {
    const int threads = TEAM == 32 ? 128 : TEAM, per = threads / TEAM;
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + per - 1) / per);
    count_launch();
    return launch_early(vec ? layer_norm_kernel<TEAM, TURNS, true> : layer_norm_kernel<TEAM, TURNS, false>, dim3(grid), threads, 0, s, a);
}

template <int TEAM, int TURNS, bool RES, int TYPE>
cudaError_t launch_stream(const LayerNormArgs& a, cudaStream_t s) {
    constexpr bool kRing = TEAM >= 512;
    constexpr int threads = TEAM <= 32 ? 128 : TEAM, per = threads / TEAM, bytes = kRing ? kRingBytes<TEAM, TURNS, RES> : 0;
    void (*kern)(LayerNormArgs);
    if constexpr (kRing)
        kern = layer_norm_ring_kernel<TEAM, TURNS, RES, TYPE>;
    else
        kern = layer_norm_stream_kernel<TEAM, TURNS, RES, TYPE>;
    static std::atomic<int> known;  // blocks that are resident at once on an SM; the same on every sm_100
    if (bytes) {
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
    count_launch();
    return launch_early(kern, dim3(static_cast<unsigned>(need < fit ? need : fit)), threads, bytes, s, a);
}
template <int TEAM, int TURNS, bool RES>
cudaError_t launch_stream(const LayerNormArgs& a, cudaStream_t s) {
    const int t = a.x_type;
    const bool one = (!a.residual || a.residual_type == t) && ((!a.weight && !a.bias) || a.weight_type == t);
    if (!one) return launch_stream<TEAM, TURNS, RES, -1>(a, s);
    return t == kTokF16 ? launch_stream<TEAM, TURNS, RES, kTokF16>(a, s) : launch_stream<TEAM, TURNS, RES, kTokBF16>(a, s);
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
