// i8_pair.cu — linear layer of 8-bit integers, many rows: tcgen05 on pairs of SMs.
//
// Bound by the tensor cores under the power limit (4096 x 4096 -> 14336 bf16: 158 to 165 us, 2.9 to 3.0 Pop/s at 1.64 GHz, 81% of
// the tensor pipe's cycles; 132 us, 3.6 Pop/s, on zeros, which take no power; 8192 x 8192 -> 8192 330 to 350 us, 3.1 to 3.3 Pop/s). Two SMs share a tile of 256 rows by up to 256 outputs (cta_group::2): each brings its 128 rows and
// half of the outputs' weights by TMA, so that an MMA of a pair reads 8 KB of each SM's shared memory in the 128 cycles that its
// 256 x 256 x 32 products take, and as much is written: what shared memory can do, where one SM alone would need half as much
// again. The accumulators are two, of 256 columns of TMEM each: the epilogue empties one while the MMAs fill the other. Pairs
// stay and walk over the tiles, rows first within groups of 16 row tiles, so that what runs at once reads the same weights.
// Few tiles of many inputs are shared by a cluster of pairs each, by ranges of the inputs (256 x 14336 -> 4096 21.5 us, 35
// without); the sum over the cluster, some 4 us, and the weights' way from memory bound those (192 x 8192 -> 8192 21.6 us).
// Ragged calls are bound by whole tiles: 1003 x 4705 -> 5003 has 128 tiles of 256 x 160 for 74 pairs, two turns (35 us).
#include "counters.hpp"
#include "i8_linear.cuh"
#include "tmap.hpp"

#include <algorithm>
#include <atomic>

namespace fxk {
namespace {

constexpr int kRows = 256;       // of a tile; each SM of the pair has half
constexpr int kMaxOutputs = 256;  // of a tile; each SM brings half of the weights
constexpr int kThreads = 320;    // warps: 0 TMA, 1 TMEM and MMA, 2..9 epilogue
constexpr int kGroup = 16;       // row tiles that are walked over before the next tile of outputs
constexpr int kLine = 256;       // bytes of results of a row that are staged where rows are not aligned
constexpr int kPitch = kLine + 16;  // with room for a line to lie as its place in memory does to a multiple of 16
constexpr int kScaleBytes = 2 * 2 * kMaxOutputs * 4, kStageBytes = 8 * 32 * kPitch;

struct Plan {
    int tile_n;  // outputs of a tile: a multiple of 32, at most 256
    int split;   // pairs of a cluster that share a tile, each with a range of the inputs; such a cluster has one tile
    int steps_each;  // steps of a pair
    int box_m;   // rows that an SM brings: 128, or fewer where there are no more
    int slots;
    int tiles_m, tiles_n;
    int scales, stage;  // offsets of the epilogue's buffers in shared memory
    int bytes;
    int y_align;  // bytes that 16 results begin at a multiple of: 32, 16, or 0 for less
};

// Loads of both SMs count their bytes on the first SM's barrier, at `bar` of the cluster's shared memory.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
// Every lane of the issuing warp runs these, on warp-uniform operands, and the one with issue != 0 executes them.
__device__ __forceinline__ void mma_i8_pair_if(uint32_t issue, uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
// Arrives on the barrier at this offset in the cluster's blocks of the mask once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair_if(uint32_t issue, uint32_t bar, uint16_t blocks) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"(blocks), "r"(issue)
        : "memory");
}
__device__ __forceinline__ uint32_t in_block(uint32_t addr, int block) {  // the same place in another block's shared memory
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(block));
    return r;
}
__device__ __forceinline__ int4 ld_cluster4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// 32 bytes to one address of a multiple of 32 (or 16, wide false).
__device__ __forceinline__ void st32(void* p, const uint32_t (&w)[8], bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    } else {
        static_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        static_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// Sixteen results one by one, the first `there` of them.
__device__ __forceinline__ void put16(uint8_t* to, int type, const float (&f)[16], int there = 16) {
    auto each = [&](auto* y, auto&& make) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < there) y[i] = make(f[i]);
    };
    if (type == kTokF32)
        each(reinterpret_cast<float*>(to), [](float v) { return v; });
    else if (type == kTokF16)
        each(reinterpret_cast<__half*>(to), [](float v) { return __float2half_rn(v); });
    else
        each(reinterpret_cast<__nv_bfloat16*>(to), [](float v) { return __float2bfloat16_rn(v); });
}
// Sixteen results to consecutive outputs.
__device__ __forceinline__ void store16(uint8_t* to, int type, const float (&f)[16], bool wide) {
    uint32_t w[8];
    if (type == kTokF32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[8 * h + i]);
            st32(to + 32 * h, w, wide);
        }
        return;
    }
    if (type == kTokF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = reinterpret_cast<const uint32_t&>(p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = reinterpret_cast<const uint32_t&>(p);
        }
    }
    st32(to, w, wide);
}

// SPLIT: the pairs of a cluster share a tile.
template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    i8_pair_kernel(const __grid_constant__ I8LinearArgs a, const __grid_constant__ Plan plan,
                   const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kI8MaxSlots + 4];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int split = SPLIT ? plan.split : 1, rank = blockIdx.x % 2, part = SPLIT ? static_cast<int>(blockIdx.x) / 2 % split : 0;
    const int pair = blockIdx.x / static_cast<uint32_t>(2 * split), pairs = gridDim.x / static_cast<uint32_t>(2 * split);  // or clusters of pairs
    const int tile_n = plan.tile_n, k_begin = part * plan.steps_each * kI8Step;
    const int steps = (min(a.k - k_begin, plan.steps_each * kI8Step) + kI8Step - 1) / kI8Step;  // at least one: the planner's split
    const uint16_t both = static_cast<uint16_t>(3 << (2 * part));  // this pair's blocks
    const int64_t tiles = static_cast<int64_t>(plan.tiles_m) * plan.tiles_n;
    const int slot_bytes = (kRows / 2 + tile_n / 2) * kI8Step;
    const uint32_t base = smem_u32(smem), bar = smem_u32(bars);
    const uint32_t full = bar, empty = bar + 8 * kI8MaxSlots, acc_full = bar + 16 * kI8MaxSlots, acc_empty = acc_full + 16;
    auto gave_up = [&](uint32_t code) {
        abort_flag = 1;
        set_status(&g_i8_status, code);
    };
    auto tile_at = [&](int64_t t, int& m, int& n) {
        const int64_t per = static_cast<int64_t>(kGroup) * plan.tiles_n, g = tiles <= per ? 0 : t / per;
        const int tall = min(kGroup, plan.tiles_m - static_cast<int>(g) * kGroup);
        const uint32_t in = static_cast<uint32_t>(t - g * per);  // below 16 * 2^23
        n = static_cast<int>(in / static_cast<uint32_t>(tall));
        m = static_cast<int>(g) * kGroup + static_cast<int>(in % static_cast<uint32_t>(tall));
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kI8MaxSlots; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 16);  // the epilogue's warps of both SMs
        }
        abort_flag = 0;
        fence_mbar_init();
    }
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&x_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&w_map) : "memory");
    }
    wait_for_earlier();  // before TMEM is taken, which the earlier kernel, of whatever library, may still ask for
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the other SM's barriers are there too
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    let_later_begin();  // TMEM is there in every block that comes here: a later kernel's blocks keep none from it

    // the epilogue's warps
    const int quad = warp % 4, half = (warp - 2) / 4, me = static_cast<int>(threadIdx.x) - 64, size = a.y_type == kTokF32 ? 4 : 2;
    const int per_line = kLine / size;  // a power of two
    float* const scales = reinterpret_cast<float*>(smem + plan.scales);  // [tile % 2][scale, bias][output]
    uint8_t* const stage = smem + plan.stage + (warp - 2) * 32 * kPitch;
    int* const partial = reinterpret_cast<int*>(smem);  // [output][row of this SM]: a cluster's sums
    const uint32_t release = in_block(acc_empty, 2 * part);
    auto row_of = [&](int m) { return static_cast<int64_t>(m) * kRows + rank * (kRows / 2) + quad * 32 + lane; };
    auto columns = [&](int first, int count, int& c_begin, int& c_end) {  // this warp's, of `count`, a multiple of 16
        const int low = (count / 16 + 1) / 2 * 16;
        c_begin = first + half * low;
        c_end = half ? first + count : first + low;
    };
    // Sixteen sums of a thread's row, from column c of the tile on, to results; c_begin and c_end: of all columns of the warp.
    auto finish16 = [&](int64_t row, int n, float xs, const float* of_tile, int c, int c_begin, int c_end, float (&f)[16]) {
        const float* const s_at = of_tile + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 sc = *reinterpret_cast<const float4*>(s_at + 4 * i);
            const float4 b = *reinterpret_cast<const float4*>(s_at + kMaxOutputs + 4 * i);
            put_pair(f, 2 * i, i8_value(pair_of(f, 2 * i), xs, make_float2(sc.x, sc.y), make_float2(b.x, b.y)));
            put_pair(f, 2 * i + 1, i8_value(pair_of(f, 2 * i + 1), xs, make_float2(sc.z, sc.w), make_float2(b.z, b.w)));
        }
        const int o0 = n * tile_n + c;
        if (plan.y_align) {
            uint8_t* const to = static_cast<uint8_t*>(a.y) + (row * a.y_stride + o0) * size;
            if (row < a.rows && o0 + 16 <= a.n)
                store16(to, a.y_type, f, plan.y_align == 32);
            else if (row < a.rows)
                put16(to, a.y_type, f, a.n - o0);
            return;
        }
        // Rows that are not aligned: up to a line of results waits in shared memory, as far behind a multiple of 16 as its
        // place in memory, and leaves in pieces of 16 bytes, which are whole but at its ends.
        const int in = (c - c_begin) & (per_line - 1), first = o0 - in;  // the line's first output
        uint8_t* const begin = static_cast<uint8_t*>(a.y) + ((row - lane) * a.y_stride + first) * size;  // of the warp's first row
        const uint32_t low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(begin)), pitch = static_cast<uint32_t>(a.y_stride) * size;
        auto behind = [&](int r) { return static_cast<int>((low + r * pitch) % 16); };
        put16(stage + lane * kPitch + behind(lane) + in * size, a.y_type, f);
        if (in + 16 != per_line && c + 16 < c_end) return;
        __syncwarp();
        const int bytes = min(in + 16, a.n - first) * size, rows = static_cast<int>(min(static_cast<int64_t>(32), a.rows - (row - lane)));
        // half a warp a row: a whole piece a lane, and a value of the ends a lane (before the first piece, behind the last)
        for (int r0 = lane / 16; r0 < 32; r0 += 8) {
            uint4 piece[4];
            uint32_t edge[4];
            int piece_at[4], edge_at[4];  // in the staged row, or -1
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = r0 + 2 * i, off = behind(r), end = r < rows ? off + max(bytes, 0) : off;
                const int head = min((off + 15) / 16 * 16, end), tail = max(end / 16 * 16, head), l = lane % 16;
                piece_at[i] = (off + 15) / 16 * 16 + 16 * l;
                if (piece_at[i] + 16 > end) piece_at[i] = -1;
                edge_at[i] = l < 8 ? off + l * size : tail + (l - 8) * size;
                if (edge_at[i] >= (l < 8 ? head : end)) edge_at[i] = -1;
                const uint8_t* const from_row = stage + r * kPitch;
                if (piece_at[i] >= 0) piece[i] = *reinterpret_cast<const uint4*>(from_row + piece_at[i]);
                if (edge_at[i] >= 0)
                    edge[i] = size == 2 ? *reinterpret_cast<const uint16_t*>(from_row + edge_at[i])
                                        : *reinterpret_cast<const uint32_t*>(from_row + edge_at[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint8_t* const to = begin + static_cast<int64_t>(r0 + 2 * i) * a.y_stride * size - behind(r0 + 2 * i);
                if (piece_at[i] >= 0) *reinterpret_cast<uint4*>(to + piece_at[i]) = piece[i];
                if (edge_at[i] < 0) continue;
                if (size == 2)
                    *reinterpret_cast<uint16_t*>(to + edge_at[i]) = static_cast<uint16_t>(edge[i]);
                else
                    *reinterpret_cast<uint32_t*>(to + edge_at[i]) = edge[i];
            }
        }
        __syncwarp();
    };

    if (warp == 0) {
        if (lane == 0) {
            int at = 0;
            uint32_t ph = 0;
            const uint32_t signal = in_block(full, 2 * part);
            for (int64_t t = pair; t < tiles && !abort_flag; t += pairs) {
                int m, n;
                tile_at(t, m, n);
                // an SM without rows brings none (what its lanes then sum up is stored nowhere)
                const int r0 = m * kRows + rank * (kRows / 2), with_rows = m * kRows + kRows / 2 < a.rows ? 2 : 1;
                const int bytes = (with_rows * plan.box_m + tile_n) * kI8Step;
                for (int step = 0; step < steps; ++step) {
                    if (!wait_phase(empty + 8 * at, ph ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                    if (abort_flag) break;
                    const uint32_t to = base + at * slot_bytes;
                    if (rank == 0) mbar_arrive_expect_tx(full + 8 * at, bytes);
                    if (r0 < a.rows) tma_load_2d_pair(to, &x_map, k_begin + step * kI8Step, r0, signal + 8 * at);
                    if (!a.hold_codes)
                        tma_load_2d_pair(to + kRows / 2 * kI8Step, &w_map, k_begin + step * kI8Step, n * tile_n + rank * (tile_n / 2),
                                         signal + 8 * at);
                    if (++at == plan.slots) at = 0, ph ^= 1;
                }
            }
            // the last slots' MMAs signal this block once more; where a role gave up, copies may still be on their way
            for (int i = 0; i < plan.slots; ++i) wait_phase(empty + 8 * i, i < at ? ph : ph ^ 1, &abort_flag, a.wait_ns);
            if (rank == 0 && abort_flag)
                for (int i = 0; i < plan.slots; ++i) wait_phase(full + 8 * i, i < at ? ph : ph ^ 1, nullptr, a.wait_ns);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = instr_desc_i8(kRows, 0) | static_cast<uint32_t>(tile_n >> 3) << 17;
            // All of TMEM is this block's, so its first column is 0, a constant that the issuing loop has at no cost; it keeps
            // to warp-uniform values throughout (and leaves at no other place than its end): a step takes the MMAs 512 cycles, and
            // one thread's own code took the loop 690 (4096 x 4096 -> 14336 165 us).
            if (tmem != 0) gave_up(kStatusBadTmem);
            const uint32_t issue = elect_one();
            int at = 0, acc = 0;
            uint32_t ph = 0, acc_ph = 0;
            for (int64_t t = pair; t < tiles; t += pairs) {
                if (!wait_phase(acc_empty + 8 * acc, acc_ph ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAccFree);
                for (int step = 0; step < steps; ++step) {
                    if (!wait_phase(full + 8 * at, ph, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
                    tc_fence_after();
                    const uint64_t ad = desc_sw128(base + at * slot_bytes), bd = ad + (kRows / 2 * kI8Step >> 4);
#pragma unroll
                    for (int i = 0; i < kI8Step / 32; ++i)
                        mma_i8_pair_if(issue, acc * kMaxOutputs, ad + 2 * i, bd + 2 * i, idesc, step > 0 || i > 0);
                    commit_pair_if(issue, empty + 8 * at, both);
                    if (++at == plan.slots) at = 0, ph ^= 1;
                }
                commit_pair_if(issue, acc_full + 8 * acc, both);
                if (++acc == 2) acc = 0, acc_ph ^= 1;
            }
            // the last MMAs end before the blocks do
            for (int i = 0; i < 2; ++i) wait_phase(acc_full + 8 * i, i < acc ? acc_ph : acc_ph ^ 1, nullptr, a.wait_ns);
        }
        __syncwarp();
    } else {
        // A thread has a row, and the two warps of a quarter's rows half of the columns each. Scales and bias of the tile's outputs
        // come to shared memory while the MMAs run. (No role leaves this loop early: its warps meet once a tile.)
        int acc = 0;
        uint32_t ph = 0;
        for (int64_t t = pair; t < tiles; t += pairs) {
            int m, n;
            tile_at(t, m, n);
            float* const of_tile = scales + acc * 2 * kMaxOutputs;
            if (me < tile_n) {
                const int o = n * tile_n + me;
                of_tile[me] = o < a.n ? a.scales[o] : 0.f;
                of_tile[kMaxOutputs + me] = o < a.n && a.bias ? a.bias[o] : -0.f;
            }
            const int64_t row = row_of(m);
            const float xs = row < a.rows ? a.x_scale[a.x_scale_mode == kScaleRow ? row : 0] : 0.f;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!wait_phase(acc_full + 8 * acc, ph, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAcc);
            __syncwarp();
            tc_fence_after();
            int c_begin, c_end;
            columns(0, tile_n, c_begin, c_end);
            const uint32_t from = tmem + acc * kMaxOutputs + (static_cast<uint32_t>(quad * 32) << 16);
            uint32_t next[16];
            tmem_ld16_nowait(from + c_begin, next);
            for (int c = c_begin; c < c_end; c += 16) {
                tmem_wait();
                tmem_regs_ready(next);
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (SPLIT)
                        partial[(c + i) * (kRows / 2) + quad * 32 + lane] = static_cast<int>(next[i]);
                    else
                        f[i] = __int2float_rn(static_cast<int>(next[i]));
                }
                if (c + 16 < c_end) tmem_ld16_nowait(from + c + 16, next);  // on its way during these columns' arithmetic
                if (!SPLIT) finish16(row, n, xs, of_tile, c, c_begin, c_end, f);
            }
            tc_fence_before();
            __syncwarp();
            // only where a later tile waits for it: no signal is on its way to a block that may have ended
            if (lane == 0 && t + 2 * static_cast<int64_t>(pairs) < tiles) arrive_cluster(release + 8 * acc);
            if (++acc == 2) acc = 0, ph ^= 1;
        }
        tc_fence_before();
    }
    if constexpr (SPLIT) {
        // The pairs of a cluster hold their sums out in shared memory, over the ring (whose MMAs are done); each adds up a share of
        // the tile's columns, 512 neighbouring bytes a warp at a time, in its own place for them, and makes results of it.
        __syncwarp();
        cluster_sync();
        const int share = tile_n / split, first = part * share * (kRows / 2) / 4;
        uint32_t from[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) from[p] = in_block(base, p < split ? 2 * p + rank : 0);
#pragma unroll 4
        for (int i = first + threadIdx.x; i < first + share * (kRows / 2) / 4; i += kThreads) {
            int4 q[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) q[p] = p < split ? ld_cluster4(from[p] + i * 16) : make_int4(0, 0, 0, 0);
            reinterpret_cast<int4*>(partial)[i] = make_int4(q[0].x + q[1].x + q[2].x + q[3].x, q[0].y + q[1].y + q[2].y + q[3].y,
                                                            q[0].z + q[1].z + q[2].z + q[3].z, q[0].w + q[1].w + q[2].w + q[3].w);
        }
        __syncthreads();
        if (warp >= 2) {
            int m, n, c_begin, c_end;
            tile_at(pair, m, n);
            const int64_t row = row_of(m);
            const float xs = row < a.rows ? a.x_scale[a.x_scale_mode == kScaleRow ? row : 0] : 0.f;
            columns(part * share, share, c_begin, c_end);
            for (int c = c_begin; c < c_end; c += 16) {
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) f[i] = __int2float_rn(partial[(c + i) * (kRows / 2) + quad * 32 + lane]);
                finish16(row, n, xs, scales, c, c_begin, c_end, f);
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (abort_flag) asm volatile("fence.acq_rel.cluster;" ::: "memory");  // signals that no one waited for
    __syncwarp();
    cluster_sync_relaxed();  // neither SM's shared memory or TMEM ends while the other may still signal or read it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

constexpr int kSmem = 226 * 1024;

// Clusters of `size` blocks that the current device runs at once.
cudaError_t clusters(int size, int* count) {
    static std::atomic<int> known[64][9];  // by device; 0: not asked yet
    int dev = 0;
    cudaGetDevice(&dev);
    *count = dev < 64 ? known[dev][size].load(std::memory_order_relaxed) : 0;
    if (*count) return cudaSuccess;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(count, i8_pair_kernel<true>, &cfg);
    if (e == cudaSuccess && dev < 64) known[dev][size].store(*count, std::memory_order_relaxed);
    return e;
}

}  // namespace

cudaError_t i8_pair_status(uint32_t* code) { return take_i8_status(code); }

cudaError_t launch_i8_pair(const I8LinearArgs& a, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(i8_pair_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(i8_pair_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    Plan p{};
    p.tiles_m = (a.rows + kRows - 1) / kRows;
    // Outputs of a tile, and pairs that share one, with the fewest cycles. A step of 32 inputs moves 256 + n lines of 32 bytes through
    // an SM's shared memory, in and out, which takes as long as the products of 256 outputs and longer than those of fewer; a
    // cluster's sum takes some 3000 cycles.
    const int pairs = sm_count() / 2, steps = (a.k + kI8Step - 1) / kI8Step;
    int64_t least = INT64_MAX;
    for (int split = 1; split <= 4; ++split) {
        int at_once = pairs;
        if (split > 1) {
            if (steps < 4 * split) break;  // with four steps a pair and at most four pairs, rounding up leaves none without a step
            if (e = clusters(2 * split, &at_once); e != cudaSuccess) return e;
        }
        for (int n = kMaxOutputs; n >= 128; n -= 32) {
            const int64_t tiles = static_cast<int64_t>(p.tiles_m) * ((a.n + n - 1) / n);
            if (split > 1 && (n % (16 * split) != 0 || tiles > at_once)) continue;
            const int64_t turns = (tiles + at_once - 1) / at_once;
            const int64_t cost = turns * ((steps + split - 1) / split) * (kRows + n) + (split > 1 ? 3000 : 0);
            if (cost < least) least = cost, p.tile_n = n, p.split = split;
        }
    }
    p.tiles_n = (a.n + p.tile_n - 1) / p.tile_n;
    p.steps_each = (steps + p.split - 1) / p.split;
    p.box_m = std::min((a.rows + 15) / 16 * 16, kRows / 2);
    const int slot = (kRows / 2 + p.tile_n / 2) * kI8Step;
    const uint64_t where = reinterpret_cast<uintptr_t>(a.y) | static_cast<uint64_t>(a.y_stride) * (a.y_type == kTokF32 ? 4 : 2);
    p.y_align = where % 32 == 0 ? 32 : where % 16 == 0 ? 16 : 0;
    const int stage = p.y_align ? 0 : kStageBytes;
    p.slots = std::min((kSmem - kScaleBytes - stage) / slot, kI8MaxSlots);
    p.scales = std::max(p.slots * slot, p.split > 1 ? kRows / 2 * p.tile_n * 4 : 0);  // a cluster's sums lie over the ring
    p.stage = p.scales + kScaleBytes;
    p.bytes = p.stage + stage;
    auto pitch = [](int64_t stride) { return (stride + 15) / 16 * 16; };  // of one row, which has none
    CUtensorMap x, w;
    e = tmap_rows(&x, a.x, 1, a.k, a.rows, pitch(a.x_stride), p.box_m);
    if (e == cudaSuccess) e = tmap_rows(&w, a.codes, 1, a.k, a.n, pitch(a.codes_stride), p.tile_n / 2);
    if (e != cudaSuccess) return e;
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * p.split * (p.split > 1 ? tiles : std::min<int64_t>(tiles, pairs))));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2 * p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, p.split > 1 ? i8_pair_kernel<true> : i8_pair_kernel<false>, a, p, x, w);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace fxk
