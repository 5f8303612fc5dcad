// i8_stream.cu — linear layer of 8-bit integers, few rows: weights stream through tcgen05.
//
// Outputs are the MMA's M, 128 a tile, and the rows of x its N, so that a weight is read once whatever the number of rows (to
// 128) and a single row costs no more than its weights: bound by memory (8 x 8192 -> 28672: 40 us, 5.9 TB/s, 90% of the copy;
// with few bytes by the launch, the first copies and a cluster's sum: 1 x 4096 -> 4096 7.2 us). TMA brings 128 inputs of both at
// a time, one warp issues the MMAs, sums are held in TMEM. Few tiles are shared by a cluster each, by ranges of the inputs;
// its blocks add up over the cluster's shared memory. Whole numbers add up to the same in any order.
#include "counters.hpp"
#include "i8_linear.cuh"
#include "tmap.hpp"

#include <algorithm>
#include <atomic>

namespace fxk {
namespace {

constexpr int kTileM = 128;
constexpr int kThreads = 192;  // warps: 0 TMA, 1 TMEM and MMA, 2..5 epilogue
// Two blocks share an SM, and never more: each has at most 256 columns of TMEM, so that none waits for another's.
constexpr int kSmemTwo = 112 * 1024, kSmemOne = 224 * 1024, kSmemLeast = 80 * 1024;

struct Plan {
    int tile_n;      // rows, rounded up to a multiple of 16: at most kI8StreamRows
    int split;       // blocks of a cluster that share a tile
    int steps_each;  // steps of a block
    int slots;
    int cols;        // of TMEM
    int bytes;
    bool y_vec;      // results aligned to four outputs
};

__global__ void __launch_bounds__(kThreads, 2)
    i8_stream_kernel(const __grid_constant__ I8LinearArgs a, const __grid_constant__ Plan plan,
                     const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kI8MaxSlots + 1];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int tile_n = plan.tile_n, split = plan.split, rank = split > 1 ? static_cast<int>(blockIdx.x) % split : 0;
    const int o0 = static_cast<int>(blockIdx.x) / split * kTileM;
    const int rows = a.rows;
    const int k_begin = rank * plan.steps_each * kI8Step;
    const int steps = (min(a.k - k_begin, plan.steps_each * kI8Step) + kI8Step - 1) / kI8Step;  // at least one: the planner's split
    const int slot_bytes = (kTileM + tile_n) * kI8Step;
    const uint32_t base = smem_u32(smem), bar = smem_u32(bars);
    const uint32_t full = bar, empty = bar + 8 * kI8MaxSlots, done = bar + 16 * kI8MaxSlots;
    auto gave_up = [&](uint32_t code) {
        abort_flag = 1;
        set_status(&g_i8_status, code);
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kI8MaxSlots; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        mbar_init(done, 1);
        abort_flag = 0;
        fence_mbar_init();
    }
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&w_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&x_map) : "memory");
    }
    wait_for_earlier();  // before TMEM is taken, which the earlier kernel, of whatever library, may still ask for
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_at), plan.cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    let_later_begin();  // TMEM is there in every block that comes here: a later kernel's blocks keep none from it

    if (warp == 0) {
        if (lane == 0) {
            int at = 0;
            uint32_t ph = 0;
            for (int step = 0; step < steps && !a.hold_codes; ++step) {
                if (!wait_phase(empty + 8 * at, ph ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                if (abort_flag) break;
                const uint32_t to = base + at * slot_bytes;
                mbar_arrive_expect_tx(full + 8 * at, slot_bytes);
                tma_load_2d(to, &w_map, k_begin + step * kI8Step, o0, full + 8 * at);
                tma_load_2d(to + kTileM * kI8Step, &x_map, k_begin + step * kI8Step, 0, full + 8 * at);
                if (++at == plan.slots) at = 0, ph ^= 1;
            }
            // copies still on their way, which roles that give up, now or later, no longer wait for
            for (int i = 0; i < plan.slots; ++i) wait_phase(full + 8 * i, i < at ? ph : ph ^ 1, nullptr, a.wait_ns);
        }
        __syncwarp();
    } else if (warp == 1) {
        // the warp as one, on uniform values: issuing from one thread's own code takes longer than short steps' MMAs
        const uint32_t idesc = instr_desc_i8(kTileM, 0) | static_cast<uint32_t>(tile_n >> 3) << 17, issue = elect_one();
        int at = 0;
        uint32_t ph = 0;
        for (int step = 0; step < steps; ++step) {
            if (!wait_phase(full + 8 * at, ph, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
            tc_fence_after();
            const uint64_t ad = desc_sw128(base + at * slot_bytes), bd = ad + (kTileM * kI8Step >> 4);
#pragma unroll
            for (int i = 0; i < kI8Step / 32; ++i) mma_i8_if(issue, tmem, ad + 2 * i, bd + 2 * i, idesc, step > 0 || i > 0);
            mma_commit_if(issue, empty + 8 * at);
            if (++at == plan.slots) at = 0, ph ^= 1;
        }
        mma_commit_if(issue, done);
        wait_phase(done, 0, nullptr, a.wait_ns);  // the epilogue may have given up: no MMA outlives its TMEM
        __syncwarp();
    } else {
        const int quad = warp % 4, row = quad * 32 + lane, out = o0 + row;
        float scale = 0.f, bias = -0.f;
        if (split == 1 && out < a.n) {
            scale = a.scales[out];
            if (a.bias) bias = a.bias[out];
        }
        if (!wait_phase(done, 0, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAcc);
        __syncwarp();
        tc_fence_after();
        const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        int* const partial = reinterpret_cast<int*>(smem);  // [row][output], over the ring
        for (int c = 0; c < tile_n; c += 16) {
            uint32_t v[16];
            tmem_ld16_nowait(acc + c, v);
            tmem_wait();
            tmem_regs_ready(v);
            if (split > 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i) partial[(c + i) * kTileM + row] = static_cast<int>(v[i]);
                continue;
            }
            const int r = c + lane % 16;
            const float xs = r < rows ? a.x_scale[a.x_scale_mode == kScaleRow ? r : 0] : 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float xi = __shfl_sync(0xffffffffu, xs, i);
                if (c + i < rows && out < a.n)
                    tok_store(a.y, static_cast<int64_t>(c + i) * a.y_stride + out, a.y_type,
                              i8_value(static_cast<int>(v[i]), xi, scale, bias));
            }
        }
        tc_fence_before();
    }
    // TMEM goes before the blocks of a cluster wait for one another: none holds it while it waits for one that may still ask for it
    __syncwarp();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, plan.cols);
    }
    if (split > 1) {  // each block adds up a share of the tile over the cluster
        __syncwarp();
        cluster_sync();
        const int all = rows * (kTileM / 4), share = (all + split - 1) / split, end = min(all, (rank + 1) * share);
        for (int i = rank * share + threadIdx.x; i < end; i += kThreads) {
            const int r = i / (kTileM / 4), o = o0 + i % (kTileM / 4) * 4;
            if (o >= a.n) continue;
            const uint32_t at = base + (r * kTileM + i % (kTileM / 4) * 4) * 4;
            int4 v[8];
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < split) v[p] = ld_cluster_s32x4(at, p);
            int s[4] = {};
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < split) s[0] += v[p].x, s[1] += v[p].y, s[2] += v[p].z, s[3] += v[p].w;
            const float xs = a.x_scale[a.x_scale_mode == kScaleRow ? r : 0];
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                f[e] = o + e < a.n ? i8_value(s[e], xs, a.scales[o + e], a.bias ? a.bias[o + e] : -0.f) : 0.f;
            i8_store4(a.y, static_cast<int64_t>(r) * a.y_stride + o, a.y_type, f, plan.y_vec && o + 4 <= a.n, a.n - o);
        }
        cluster_sync();  // no block's shared memory ends while another reads it
    }
}

// Clusters of `size` blocks that the current device runs at once, with shared memory for one or two blocks an SM.
cudaError_t clusters(int size, bool two, int* count) {
    static std::atomic<int> known[64][2][9];  // by device; 0: not asked yet
    int dev = 0;
    cudaGetDevice(&dev);
    *count = dev < 64 ? known[dev][two][size].load(std::memory_order_relaxed) : 0;
    if (*count) return cudaSuccess;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = two ? kSmemTwo : kSmemOne;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(count, i8_stream_kernel, &cfg);
    if (e == cudaSuccess && dev < 64) known[dev][two][size].store(*count, std::memory_order_relaxed);
    return e;
}

}  // namespace

cudaError_t i8_stream_status(uint32_t* code) { return take_i8_status(code); }

cudaError_t launch_i8_stream(const I8LinearArgs& a, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(i8_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOne);
    if (e != cudaSuccess) return e;
    Plan p{};
    if (a.rows > kI8StreamRows) return cudaErrorInvalidValue;
    p.tile_n = (a.rows + 15) / 16 * 16;
    const int tiles = (a.n + kTileM - 1) / kTileM, all_steps = (a.k + kI8Step - 1) / kI8Step;
    const int slot = (kTileM + p.tile_n) * kI8Step;
    // Up to 64 rows two blocks share an SM, so that one's copies go on while the other begins or ends; more rows need the shared
    // memory for copies on their way (128 x 4096 -> 4096 11 us, 12.1 with two; 64 rows 9.5 us, 9.9 with one).
    const bool two = p.tile_n <= 64;
    int split = 1;
    for (int c = 8; c > 1 && split == 1; --c) {
        if (all_steps < 2 * c || tiles * c > sm_count() * (two ? 2 : 1)) continue;
        int most = 0;
        if (e = clusters(c, two, &most); e != cudaSuccess) return e;
        if (tiles <= most) split = c;
    }
    p.steps_each = (all_steps + split - 1) / split;
    p.split = (all_steps + p.steps_each - 1) / p.steps_each;  // no block without a step
    const int room = two ? kSmemTwo : kSmemOne;
    p.slots = std::min({room / slot, kI8MaxSlots, std::max(p.steps_each, 2)});
    p.bytes = std::max({p.slots * slot, p.split > 1 ? p.tile_n * kTileM * 4 : 0, kSmemLeast});
    p.cols = 32;
    while (p.cols < p.tile_n) p.cols *= 2;
    const int64_t unit = a.y_type == kTokF32 ? 16 : 8;
    p.y_vec = reinterpret_cast<uintptr_t>(a.y) % unit == 0 && a.y_stride % 4 == 0;
    auto pitch = [](int64_t stride) { return (stride + 15) / 16 * 16; };  // of one row, which has none
    CUtensorMap w, x;
    e = tmap_rows(&w, a.codes, 1, a.k, a.n, pitch(a.codes_stride), kTileM);
    if (e == cudaSuccess) e = tmap_rows(&x, a.x, 1, a.k, a.rows, pitch(a.x_stride), p.tile_n);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * p.split);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, i8_stream_kernel, a, p, w, x);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace fxk
