// i8_pair.cu — linear layer of 8-bit integers, many rows: tcgen05 on pairs of SMs.
//
// Bound by the tensor cores. Two SMs share a tile of 256 rows by up to 256 outputs (cta_group::2): each brings its 128 rows and
// half of the outputs' weights by TMA, so that an MMA of a pair reads 8 KB of each SM's shared memory in the 128 cycles that its
// 256 x 256 x 32 products take, and as much is written: what shared memory can do, where one SM alone would need half as much
// again. The accumulators are two, of 256 columns of TMEM each: the epilogue empties one while the MMAs fill the other. Pairs
// stay and walk over the tiles, rows first within groups of 16 row tiles, so that what runs at once reads the same weights.
#include "counters.hpp"
#include "i8_linear.cuh"
#include "tmap.hpp"

#include <algorithm>
#include <atomic>

namespace fxk {
namespace {

constexpr int kRows = 256;       // of a tile; each SM of the pair has half
constexpr int kMaxOutputs = 256;  // of a tile; each SM brings half of the weights
constexpr int kThreads = 192;    // warps: 0 TMA, 1 TMEM and MMA, 2..5 epilogue
constexpr int kGroup = 16;       // row tiles that are walked over before the next tile of outputs
constexpr int kPitch = 36;       // words of a staged row of 32 sums

struct Plan {
    int tile_n;  // outputs of a tile: a multiple of 32, at most 256
    int slots;
    int tiles_m, tiles_n;
    int stage;  // offset of the epilogue's buffers in shared memory
    int bytes;
    bool y_vec;  // results aligned to four outputs
};

// Loads of both SMs count their bytes on the first SM's barrier, at `bar` of the cluster's shared memory.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on the barrier at this offset in both SMs once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}
__device__ __forceinline__ uint32_t of_first(uint32_t addr) {  // the same place in the first SM's shared memory
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__global__ void __launch_bounds__(kThreads, 1)
    i8_pair_kernel(const __grid_constant__ I8LinearArgs a, const __grid_constant__ Plan plan,
                   const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kI8MaxSlots + 4];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = blockIdx.x % 2, pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    const int tile_n = plan.tile_n, steps = (a.k + kI8Step - 1) / kI8Step;
    const int64_t tiles = static_cast<int64_t>(plan.tiles_m) * plan.tiles_n;
    const int slot_bytes = (kRows / 2 + tile_n / 2) * kI8Step;
    const uint32_t base = smem_u32(smem), bar = smem_u32(bars);
    const uint32_t full = bar, empty = bar + 8 * kI8MaxSlots, acc_full = bar + 16 * kI8MaxSlots, acc_empty = acc_full + 16;
    auto gave_up = [&](uint32_t code) {
        abort_flag = 1;
        set_status(&g_i8_status, code);
    };
    auto tile_at = [&](int64_t t, int& m, int& n) {
        const int64_t per = static_cast<int64_t>(kGroup) * plan.tiles_n, g = t / per, in = t - g * per;
        const int tall = min(kGroup, plan.tiles_m - static_cast<int>(g) * kGroup);
        n = static_cast<int>(in / tall);
        m = static_cast<int>(g) * kGroup + static_cast<int>(in % tall);
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kI8MaxSlots; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 8);  // the epilogue's warps of both SMs
        }
        abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the other SM's barriers are there too
    tc_fence_after();
    const uint32_t tmem = tmem_at;

    if (warp == 0) {
        if (lane == 0) {
            int at = 0;
            uint32_t ph = 0;
            const uint32_t signal = of_first(full);
            for (int64_t t = pair; t < tiles && !abort_flag; t += pairs) {
                int m, n;
                tile_at(t, m, n);
                for (int step = 0; step < steps; ++step) {
                    if (!wait_phase(empty + 8 * at, ph ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                    if (abort_flag) break;
                    const uint32_t to = base + at * slot_bytes;
                    if (rank == 0) mbar_arrive_expect_tx(full + 8 * at, 2 * slot_bytes);
                    tma_load_2d_pair(to, &x_map, step * kI8Step, m * kRows + rank * (kRows / 2), signal + 8 * at);
                    if (!a.hold_codes)
                        tma_load_2d_pair(to + kRows / 2 * kI8Step, &w_map, step * kI8Step, n * tile_n + rank * (tile_n / 2), signal + 8 * at);
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
        if (rank == 0 && lane == 0) {
            const uint32_t idesc = instr_desc_i8(kRows, 0) | static_cast<uint32_t>(tile_n >> 3) << 17;
            int at = 0, acc = 0;
            uint32_t ph = 0, acc_ph = 0;
            for (int64_t t = pair; t < tiles && !abort_flag; t += pairs) {
                if (!wait_phase(acc_empty + 8 * acc, acc_ph ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAccFree);
                tc_fence_after();
                const uint32_t d = tmem + acc * kMaxOutputs;
                for (int step = 0; step < steps; ++step) {
                    if (!wait_phase(full + 8 * at, ph, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
                    if (abort_flag) break;
                    tc_fence_after();
                    const uint64_t ad = desc_sw128(base + at * slot_bytes), bd = desc_sw128(base + at * slot_bytes + kRows / 2 * kI8Step);
#pragma unroll
                    for (int i = 0; i < kI8Step / 32; ++i) mma_i8_pair(d, ad + 2 * i, bd + 2 * i, idesc, step > 0 || i > 0);
                    commit_pair(empty + 8 * at);
                    if (++at == plan.slots) at = 0, ph ^= 1;
                }
                commit_pair(acc_full + 8 * acc);
                if (++acc == 2) acc = 0, acc_ph ^= 1;
            }
            // the last MMAs end before the blocks do
            for (int i = 0; i < 2; ++i) wait_phase(acc_full + 8 * i, i < acc ? acc_ph : acc_ph ^ 1, nullptr, a.wait_ns);
        }
        __syncwarp();
    } else {
        // 32 columns at a time: a thread reads its row's sums, which change places in shared memory, so that a store is four
        // outputs (or one) of neighbours
        const int quad = warp % 4;
        int* const stage = reinterpret_cast<int*>(smem + plan.stage) + quad * 32 * kPitch;
        const uint32_t release = of_first(acc_empty);
        int acc = 0;
        uint32_t ph = 0;
        for (int64_t t = pair; t < tiles; t += pairs) {
            int m, n;
            tile_at(t, m, n);
            const int r0 = m * kRows + rank * (kRows / 2) + quad * 32;
            const float xs = r0 + lane < a.rows ? a.x_scale[a.x_scale_mode == kScaleRow ? r0 + lane : 0] : 0.f;
            const int rows = min(32, a.rows - r0);  // of this warp; none or fewer where the tile is ragged
            if (!wait_phase(acc_full + 8 * acc, ph, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAcc);
            if (__any_sync(0xffffffffu, abort_flag)) break;
            tc_fence_after();
            const uint32_t from = tmem + acc * kMaxOutputs + (static_cast<uint32_t>(quad * 32) << 16);
            for (int c = 0; c < tile_n; c += 32) {
                uint32_t v[2][16];
                tmem_ld16_nowait(from + c, v[0]);
                tmem_ld16_nowait(from + c + 16, v[1]);
                tmem_wait();
                tmem_regs_ready(v[0]);
                tmem_regs_ready(v[1]);
                __syncwarp();  // the columns before these have left the buffer
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<uint4*>(stage + lane * kPitch + 4 * i) =
                        make_uint4(v[i / 4][4 * (i % 4)], v[i / 4][4 * (i % 4) + 1], v[i / 4][4 * (i % 4) + 2], v[i / 4][4 * (i % 4) + 3]);
                __syncwarp();
                const int o0 = n * tile_n + c;
                if (plan.y_vec && o0 + 32 <= a.n) {
                    const int o = o0 + lane % 8 * 4;
                    float sc[4], b[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[e] = __ldg(a.scales + o + e);
                        b[e] = a.bias ? __ldg(a.bias + o + e) : -0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = i * 4 + lane / 8;
                        const float x = __shfl_sync(0xffffffffu, xs, r);
                        const int4 s = *reinterpret_cast<const int4*>(stage + r * kPitch + lane % 8 * 4);
                        const float f[4] = {i8_value(s.x, x, sc[0], b[0]), i8_value(s.y, x, sc[1], b[1]),
                                            i8_value(s.z, x, sc[2], b[2]), i8_value(s.w, x, sc[3], b[3])};
                        if (r < rows) i8_store4(a.y, static_cast<int64_t>(r0 + r) * a.y_stride + o, a.y_type, f, true, 4);
                    }
                } else {
                    const int o = o0 + lane;
                    const float sc = o < a.n ? __ldg(a.scales + o) : 0.f, b = o < a.n && a.bias ? __ldg(a.bias + o) : -0.f;
#pragma unroll 8
                    for (int r = 0; r < 32; ++r) {
                        const float x = __shfl_sync(0xffffffffu, xs, r);
                        if (r < rows && o < a.n)
                            tok_store(a.y, static_cast<int64_t>(r0 + r) * a.y_stride + o, a.y_type, i8_value(stage[r * kPitch + lane], x, sc, b));
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(release + 8 * acc);
            if (++acc == 2) acc = 0, ph ^= 1;
        }
        tc_fence_before();
    }
    __syncwarp();
    __syncthreads();
    cluster_sync();  // neither SM's shared memory or TMEM ends while the other may still signal or read it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace

cudaError_t i8_pair_status(uint32_t* code) { return take_i8_status(code); }

cudaError_t launch_i8_pair(const I8LinearArgs& a, cudaStream_t s) {
    constexpr int kSmem = 226 * 1024;
    cudaError_t e = cudaFuncSetAttribute(i8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    Plan p{};
    p.tiles_m = (a.rows + kRows - 1) / kRows;
    // Outputs of a tile: the number whose turns over the pairs cost least. A step of 32 inputs moves 256 + n lines of 32 bytes
    // through an SM's shared memory, in and out, which takes as long as the products of 256 outputs and longer than those of
    // fewer.
    const int pairs = sm_count() / 2;
    int64_t least = INT64_MAX;
    for (int n = kMaxOutputs; n >= 128; n -= 32) {
        const int64_t tiles = static_cast<int64_t>(p.tiles_m) * ((a.n + n - 1) / n), cost = (tiles + pairs - 1) / pairs * (kRows + n);
        if (cost < least) least = cost, p.tile_n = n;
    }
    p.tiles_n = (a.n + p.tile_n - 1) / p.tile_n;
    const int slot = (kRows / 2 + p.tile_n / 2) * kI8Step, stage = 4 * 32 * kPitch * 4;
    p.slots = std::min((kSmem - stage) / slot, kI8MaxSlots);
    p.stage = p.slots * slot;
    p.bytes = p.stage + stage;
    const int64_t unit = a.y_type == kTokF32 ? 16 : 8;
    p.y_vec = reinterpret_cast<uintptr_t>(a.y) % unit == 0 && a.y_stride % 4 == 0;
    auto pitch = [](int64_t stride) { return (stride + 15) / 16 * 16; };  // of one row, which has none
    CUtensorMap x, w;
    e = tmap_rows(&x, a.x, 1, a.k, a.rows, pitch(a.x_stride), kRows / 2);
    if (e == cudaSuccess) e = tmap_rows(&w, a.codes, 1, a.k, a.n, pitch(a.codes_stride), p.tile_n / 2);
    if (e != cudaSuccess) return e;
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(tiles, pairs)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, i8_pair_kernel, a, p, x, w);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace fxk
