// w4_many.cuh — linear layer with 4-bit weights and group scales, many rows: tcgen05.
//
// A tile is 256 outputs by up to 192 rows, or 128 by up to 256; outputs are the MMA's M, rows its N. Codes come by
// TMA; sixteen warps turn them into 16-bit weights and put them into TMEM, from where the MMAs take their A operand:
// shared memory, which an MMA of M = 128 already reads for its B operand at half its bandwidth, is spared a write and
// a read of every weight. Two tiles of 128 outputs share each B operand, for the same reason and for the L2's. The
// rows come by TMA as they are (or, for e4m3 and unaligned rows, through four loader warps); one thread issues the
// MMAs, which accumulate in TMEM in f32. Few tiles share a cluster each, by ranges of k, and add up over its shared
// memory.
// Bounds: with many rows the tensor cores under the power limit, whose clock goes with the operands and the GPU's heat
// (4096 x 4096 -> 14336 bf16: 353 us on uniform codes, 1.36 PFLOP/s, 99% of a sustained library product's rate; 359 on
// normal weights, up to 411 with other rows each time and between other work, 1.17 PFLOP/s); up to 64 rows the making of weights, some two
// instructions a weight on pipes of half rate (64 x 4096 -> 14336: 20 us, as long as 16 rows take); with e4m3 rows
// their widening (4096 rows 486 to 585 us).
// A weight scale * (code - zero) is rounded once to the rows' 16-bit type (f16 for e4m3 rows): code - zero is
// exact, and the scale enters as the sum of two 16-bit values, one product and one fused multiply-add. In f16
// each output's weights are divided by the power of two below its largest scale, so that no scale's size
// overflows the type or sinks below it; the epilogue multiplies by it again.
// f16 results of bf16 rows hold eight times finer steps than bf16 weights: there a weight is the sum of two bf16 values,
// right to 2^-15 of it, each multiplied by the rows in an MMA of its own (root mean square error 2.1e-4 of the result's
// size, f16's own rounding, 1.7e-3 with one term; 64 x 4096 -> 14336 27 us, 20 with one; 4096 rows 605 and 354).
#pragma once

#include "counters.hpp"
#include "ptx.cuh"
#include "tmap.hpp"
#include "token.cuh"
#include "w4.cuh"

namespace fxk {
namespace {

// K-major operand rows of 128 bytes, 128-byte swizzle: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | static_cast<uint64_t>(1) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

// D[tmem] (+)= A[tmem] * B[smem desc]^T, 16-bit inputs, f32 accumulate: every lane runs the code, on warp-uniform
// operands, and the lane with issue != 0 executes it.
__device__ __forceinline__ void mma_f16_ta_if(uint32_t issue, uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
// Eight 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four f32 of a block of the cluster, at a shared-memory address of this one.
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, int rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\tld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [r];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr), "r"(rank));
    return v;
}

template <bool BF>
__device__ __forceinline__ uint32_t pair16(float a, float b) {
    if (BF) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return reinterpret_cast<uint32_t&>(h);
    }
    __half2 h = __floats2half2_rn(a, b);
    return reinterpret_cast<uint32_t&>(h);
}
// A 16-bit value's bits (the low half) as f32.
__device__ __forceinline__ float value16(uint32_t bits, bool is_f16) {
    return is_f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(bits))) : __uint_as_float(bits << 16);
}
template <bool BF>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF)
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    if (BF)
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    else
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

// Codes (2 i, 2 i + 1) of a word of eight as 16-bit floats code - zero, in their order; z from zero_terms.
template <bool BF>
__device__ __forceinline__ uint32_t code_pair_in_order(uint32_t w, uint32_t w4, int i, uint32_t z) {
    uint32_t r;
    if (BF) {  // 128 + code: the second code from the word shifted by four
        const uint32_t v = and_or(__byte_perm(w, w4, 0x0000 + i + ((4 + i) << 8)), 0x000f000fu, 0x43004300u);
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(z));
        return r;
    }
    // 1024 + code and 1024 + 16 code, times 1 and 1/16, less 1024 + zero and 64 + zero
    const uint32_t v = and_or(__byte_perm(w, 0, 0x4040 + i + (i << 8)), 0x00f0000fu, 0x64006400u);
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0x2c003c00u), "r"(z));
    return r;
}
template <bool BF>
__device__ __forceinline__ uint32_t zero_terms(uint32_t zero) {
    if (BF) return 0x43004300u + 0x00010001u * zero;
    return 0xd400e400u + 0x00100001u * zero;  // -(64 + zero), -(1024 + zero)
}

// 16 codes (two words) under one scale as eight pairs of weights.
template <bool BF, bool EX>
__device__ __forceinline__ void weights16(uint32_t w0, uint32_t w1, uint32_t hi, uint32_t lo, uint32_t z, uint32_t (&out)[8]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint32_t w = c ? w1 : w0, w4 = BF ? w >> 4 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = code_pair_in_order<BF>(w, w4, i, z);
            out[4 * c + i] = EX ? mul2<BF>(v, hi) : fma2<BF>(v, hi, mul2<BF>(v, lo));
        }
    }
}

// The same as the sum of two 16-bit values: the weight rounded, and what that left (exact where EX).
template <bool BF, bool EX>
__device__ __forceinline__ void weight_terms16(uint32_t w0, uint32_t w1, uint32_t hi, uint32_t lo, uint32_t z,
                                               uint32_t (&out)[8], uint32_t (&rest)[8]) {
    weights16<BF, EX>(w0, w1, hi, lo, z, out);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint32_t w = c ? w1 : w0, w4 = BF ? w >> 4 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = code_pair_in_order<BF>(w, w4, i, z), left = fma2<BF>(v, hi, out[4 * c + i] ^ 0x80008000u);
            rest[4 * c + i] = EX ? left : fma2<BF>(v, lo, left);
        }
    }
}

// Warps: 0..15 weights and epilogue, 16 codes by TMA, 17 MMA and TMEM, 18 rows by TMA, or 18..21 rows
// that have to be widened or loaded.
// TWO: 256 outputs a tile in two accumulators, else 128.
constexpr int kMakers = 16;

// TMA: the rows come as they are, else four warps write them. SS: steps of 64 inputs that share a slot of the rows' ring (a
// constant: the issuing thread has no time to spare).
// CH: scales of a step of 64 inputs (1: groups are multiples of 64). EX: the scales' type is the
// operands', so that they have no second term (in f16 but for those 2^14 below their output's largest, whose last bits
// are 2^-25 of it). TERMS: a weight is two terms.
template <bool BF, bool TWO, bool TMA, int SS, int CH, bool EX, bool TERMS>
__global__ void __launch_bounds__(TMA ? 608 : 704, 1)
    w4_many_kernel(const __grid_constant__ W4LinearArgs a, const __grid_constant__ ManyPlan plan,
                   const __grid_constant__ CUtensorMap codes_map, const __grid_constant__ CUtensorMap rows_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[7 * kMaxRing + 1];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int abort_flag;
    static_assert(!(TWO && TERMS), "two blocks of weights a step at most");
    constexpr int kTileM = TWO ? 256 : 128, kWeightCols = TWO || TERMS ? 64 : 32;  // of a step
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int n = a.w.n, k = a.w.k, group = a.w.group, groups = k / group;
    const int tile_n = plan.tile_n, rank = plan.split > 1 ? static_cast<int>(blockIdx.x) % plan.split : 0;
    const int o0 = static_cast<int>(blockIdx.x) / plan.split * kTileM;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * tile_n;
    const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows) - r0, static_cast<int64_t>(tile_n)));
    const int k_begin = rank * plan.stages_each * kStageK, k_end = min(k, k_begin + plan.stages_each * kStageK);
    const int stages = (k_end - k_begin + kStageK - 1) / kStageK;  // at least one: the planner's split
    const int steps = (k_end - k_begin + kStepK - 1) / kStepK;
    const uint32_t bar = smem_u32(bars);
    const uint32_t c_full = bar, c_empty = bar + 8 * kMaxRing, w_full = bar + 16 * kMaxRing, w_empty = bar + 24 * kMaxRing,
                   x_full = bar + 32 * kMaxRing, x_empty = bar + 40 * kMaxRing, raw_full = bar + 48 * kMaxRing,
                   done = bar + 56 * kMaxRing;
    const uint32_t codes = smem_u32(smem + plan.codes), xrows = smem_u32(smem + plan.rows);
    auto gave_up = [&](uint32_t code) {
        abort_flag = 1;
        set_w4_status(code);
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxRing; ++i) {
            mbar_init(c_full + 8 * i, 1);
            mbar_init(c_empty + 8 * i, kMakers);
            mbar_init(w_full + 8 * i, TWO ? 8 : 4);
            mbar_init(w_empty + 8 * i, 1);
            mbar_init(x_full + 8 * i, TMA ? 1 : SS);  // SS warps write a slot
            mbar_init(raw_full + 8 * i, 1);
            mbar_init(x_empty + 8 * i, 1);
        }
        mbar_init(done, 1);
        abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 17) {
        tmem_alloc(smem_u32(&tmem_at), plan.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at, weights = tmem + plan.weight_col;

    if (warp == 16) {
        if (lane == 0) {
            int cs = 0;
            uint32_t cp = 0;
            for (int st = 0; st < stages && !a.hold_codes; ++st) {
                if (!wait_phase(c_empty + 8 * cs, cp ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                if (abort_flag) break;
                mbar_arrive_expect_tx(c_full + 8 * cs, kTileM * 128);
                tma_load_2d(codes + cs * kTileM * 128, &codes_map, (k_begin + st * kStageK) / 16, o0, c_full + 8 * cs);
                if (++cs == plan.rings[0]) cs = 0, cp ^= 1;
            }
            // copies still on their way, which roles that give up, now or later, no longer wait for
            for (int i = 0; i < plan.rings[0]; ++i) wait_phase(c_full + 8 * i, (i < cs ? cp : cp ^ 1), nullptr, a.wait_ns);
        }
        __syncwarp();
    } else if (TMA && warp == 18) {  // not the codes' thread: neither ring's waits hold up the other
        if (lane == 0) {
            int xs = 0;
            uint32_t xp = 0;
            for (int step = 0; step < steps; step += SS) {
                const int boxes = min(SS, steps - step);
                if (!wait_phase(x_empty + 8 * xs, xp ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                if (abort_flag) break;
                mbar_arrive_expect_tx(x_full + 8 * xs, boxes * tile_n * 128);
                for (int i = 0; i < boxes; ++i)
                    tma_load_2d(xrows + (xs * SS + i) * tile_n * 128, &rows_map, k_begin + (step + i) * kStepK,
                                static_cast<int>(r0), x_full + 8 * xs);
                if (++xs == plan.rings[2]) xs = 0, xp ^= 1;
            }
            for (int i = 0; i < plan.rings[2]; ++i) wait_phase(x_full + 8 * i, (i < xs ? xp : xp ^ 1), nullptr, a.wait_ns);
        }
        __syncwarp();
    } else if (warp == 17) {
        const uint32_t idesc = instr_desc(128, 0, BF ? kOpBF16 : kOpF16) | static_cast<uint32_t>(tile_n >> 3) << 17;
        // All of TMEM is this block's, so its first column is 0, a constant that the issuing loop has at no cost; it keeps
        // to warp-uniform values throughout, as its own time bounds short steps.
        if (tmem != 0) gave_up(kStatusBadTmem);
        const uint32_t issue = elect_one();
        int ws = 0, xs = 0, x_step = 0;
        uint32_t wp = 0, xp = 0;
        for (int step = 0; step < steps; ++step) {
            if (x_step == 0 && !wait_phase(x_full + 8 * xs, xp, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
            if (!wait_phase(w_full + 8 * ws, wp, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
            tc_fence_after();
            const uint64_t bd = desc_sw128(xrows + (xs * SS + x_step) * tile_n * 128);
#pragma unroll
            for (int m = 0; m < kWeightCols / 32; ++m) {
                const uint32_t ad = plan.weight_col + ws * kWeightCols + m * 32;
#pragma unroll
                for (int i = 0; i < kStepK / 16; ++i)
                    mma_f16_ta_if(issue, TWO ? m * tile_n : 0, ad + 8 * i, bd + 2 * i, idesc,
                                  step > 0 || i > 0 || (TERMS && m > 0));
            }
            mma_commit_if(issue, w_empty + 8 * ws);
            if (++ws == plan.rings[1]) ws = 0, wp ^= 1;
            if (++x_step == SS || step == steps - 1) {
                mma_commit_if(issue, x_empty + 8 * xs);
                x_step = 0;
                if (++xs == plan.rings[2]) xs = 0, xp ^= 1;
            }
        }
        mma_commit_if(issue, done);
        wait_phase(done, 0, nullptr, a.wait_ns);  // the epilogue may have given up: no MMA outlives its TMEM
    } else if (!TMA && warp >= 18) {
        // rows that TMA does not bring as they are used: four warps write them in 16-byte cells of eight values, as the
        // swizzle places them
        // (a step each, so that a step's latency is hidden behind the others')
        static_assert(kRowWarps % SS == 0, "a slot is written in one turn of the warps");
        const int tid = threadIdx.x - 18 * 32, kxb = a.x_type == kTokE4M3 ? 1 : 2;
        auto fetch = [&](int step, int slot) {  // e4m3: TMA brings 128 inputs at a time, these warps widen them
            if (step < steps) {
                mbar_arrive_expect_tx(raw_full + 8 * slot, tile_n * 128);
                tma_load_2d(smem_u32(smem + plan.raw) + slot * tile_n * 128, &rows_map, (k_begin + step * kStepK) / 8,
                            static_cast<int>(r0), raw_full + 8 * slot);
            }
        };
        if (tid == 0)
            for (int i = 0; i < plan.raw_slots; ++i) fetch(2 * i, i);
        for (int step0 = 0; step0 < steps; step0 += kRowWarps) {
            const int step = step0 + tid / 32, pair = step / 2, slots = plan.raw_slots ? plan.raw_slots : 1, rs = pair % slots;
            // (the warp that shares its raw slot has asked for the last one)
            if (SS < kRowWarps && step / SS * SS >= steps) break;
            const int xs = step / SS % plan.rings[2];
            const uint32_t xp = step / SS / plan.rings[2] & 1, rp = pair / slots & 1;
            if (!wait_phase(x_empty + 8 * xs, xp ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
            uint8_t* const to = smem + plan.rows + (xs * SS + step % SS) * tile_n * 128;
            if (step < steps && plan.raw_slots) {
                if (!wait_phase(raw_full + 8 * rs, rp, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
                // eight lanes take a cell of eight rows each: every bank once, read and written
                const int at = lane % 8, c = lane / 8;
                const uint8_t* const raw = smem + plan.raw + rs * tile_n * 128 + at * 128 + (((4 * (step % 2) + c) ^ at) << 4);
                uint8_t* const lo = to + at * 128 + (((2 * c) ^ at) << 4);
                uint8_t* const hi = to + at * 128 + (((2 * c + 1) ^ at) << 4);
#pragma unroll 4
                for (int r = 0; r < tile_n * 128; r += 1024) {
                    const uint4 v = *reinterpret_cast<const uint4*>(raw + r);
                    *reinterpret_cast<uint4*>(lo + r) = widened(v, kTokE4M3);
                    *reinterpret_cast<uint4*>(hi + r) = widened(make_uint4(v.z, v.w, 0, 0), kTokE4M3);
                }
            } else if (step < steps) {
                const int k0 = k_begin + step * kStepK;
                const uint8_t* const src = static_cast<const uint8_t*>(a.x) + (r0 * a.x_stride + k0) * kxb;
#pragma unroll 2
                for (int i = lane; i < tile_n * 8; i += 32) {
                    const int r = i / 8, c = i % 8;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (r < rows && k0 + c * 8 < k_end)
                        v = raw_eight(src + (static_cast<int64_t>(r) * a.x_stride + c * 8) * kxb, a.x_type, plan.x_vec);
                    *reinterpret_cast<uint4*>(to + r * 128 + ((c ^ (r & 7)) << 4)) = widened(v, a.x_type);
                }
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(x_full + 8 * xs);
            // another use: both warps are done with the raw slot
            if (plan.raw_slots && pair * 2 + 2 * plan.raw_slots < steps) {
                asm volatile("bar.sync %0, 64;" ::"r"(2 + tid / 64) : "memory");
                if (tid % 64 == 0) fetch(pair * 2 + 2 * plan.raw_slots, rs);
            }
        }
        __syncwarp();
        if (abort_flag)  // copies still on their way: either phase may be the last that was asked for
            for (int i = 0; i < plan.raw_slots; ++i) {
                wait_phase(raw_full + 8 * i, 0, nullptr, a.wait_ns);
                wait_phase(raw_full + 8 * i, 1, nullptr, a.wait_ns);
            }
    } else {
        // a thread makes weights of one output, whose TMEM lane is its own; the four warps of a lane quarter take the steps
        // in turn (with two tiles, two warps a tile), so that a step's latency is hidden behind the others'
        constexpr int kSets = TWO ? 2 : 4;
        const int quad = warp % 4, part = warp / 4, set = part % kSets, row = (TWO ? part / 2 * 128 : 0) + quad * 32 + lane;
        const int64_t at = static_cast<int64_t>(min(o0 + row, n - 1)) * groups;
        const bool wide = a.w.scale_type == kTokF32, is_f16 = a.w.scale_type == kTokF16;
        auto scale_at = [&](int g) { return tok_load(a.w.scales, at + g, a.w.scale_type); };
        float back = 1.f, factor = 1.f;  // the output's power of two, and its reciprocal
        if (!BF) {
            // the warps of a lane quarter look through a share of the scales each
            uint32_t* const tops = reinterpret_cast<uint32_t*>(smem + plan.tops);
            if (set == 0) tops[row] = 0;
            asm volatile("bar.sync 1, %0;" ::"n"(kMakers * 32) : "memory");
            float top = 0.f;
            const uint8_t* const p = static_cast<const uint8_t*>(a.w.scales) + at * (wide ? 4 : 2);
            if (!wide && groups % 8 == 0 && reinterpret_cast<uintptr_t>(a.w.scales) % 16 == 0) {
#pragma unroll 4
                for (int g = set * 8; g < groups; g += kSets * 8) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + g * 2));
                    const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        top = fmaxf(top, value16((i % 2 ? r[i / 2] >> 16 : r[i / 2]) & 0x7fffu, is_f16));
                    }
                }
            } else {
#pragma unroll 8
                for (int g = set; g < groups; g += kSets) top = fmaxf(top, fabsf(scale_at(g)));
            }
            atomicMax(tops + row, __float_as_uint(top));  // of numbers that are not negative the bits are in order
            asm volatile("bar.sync 1, %0;" ::"n"(kMakers * 32) : "memory");
            top = __uint_as_float(tops[row]);
            // 2^e <= top < 2^(e + 1), e kept where 2^e and 2^-e are normal; an infinity or zero keeps 1
            if (top > 0.f && top < INFINITY) {
                const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
                back = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                factor = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            }
        }
        // scales, as they are stored, and zero points of a stage's steps, a stage ahead
        constexpr int kMine = kStageK / kStepK / kSets;
        uint32_t sc[kMine][CH], zo[kMine][CH];
        const float inv_group = 1.f / static_cast<float>(group);
        const uint8_t* const s_at = static_cast<const uint8_t*>(a.w.scales) + at * (wide ? 4 : 2);
        const uint8_t* const z_at = a.w.zeros ? a.w.zeros + at : nullptr;
        auto load_scales = [&](int k0) {
#pragma unroll
            for (int c = 0; c < kMine; ++c)
#pragma unroll
                for (int h = 0; h < CH; ++h) {
                    const int kc = k0 + (c * kSets + set) * kStepK + h * 32;
                    sc[c][h] = 0;  // past the end weights are zeros
                    zo[c][h] = 8;
                    if (kc < k_end) {
                        // (kc + 1/2) / group truncated: exact while k < 2^21
                        const int g =
                            k < (1 << 21) ? static_cast<int>((static_cast<float>(kc) + 0.5f) * inv_group) : kc / group;
                        if (wide)
                            sc[c][h] = __ldg(reinterpret_cast<const uint32_t*>(s_at) + g);
                        else
                            sc[c][h] = __ldg(reinterpret_cast<const uint16_t*>(s_at) + g);
                        if (z_at) zo[c][h] = __ldg(z_at + g);
                    }
                }
        };
        load_scales(k_begin);
        const uint32_t to = weights + (TWO ? part / 2 * 32 : 0) + (static_cast<uint32_t>(quad * 32) << 16);
        int cs = 0, ws = set, step = set;
        uint32_t cp = 0, wp = 0;
        for (int st = 0; st < stages; ++st) {
            uint32_t hi[kMine][CH], lo[kMine][CH], z[kMine][CH];
#pragma unroll
            for (int c = 0; c < kMine; ++c)
#pragma unroll
                for (int h = 0; h < CH; ++h) {
                    const uint32_t raw = sc[c][h];
                    float v = wide ? __uint_as_float(raw) : value16(raw, is_f16);
                    if (!BF) v *= factor;
                    hi[c][h] = pair16<BF>(v, v);
                    if (!EX) {
                        const float l = v - value16(hi[c][h], !BF);
                        lo[c][h] = fabsf(l) < INFINITY ? pair16<BF>(l, l) : 0;  // an infinite scale has no remainder
                    }
                    z[c][h] = zero_terms<BF>(zo[c][h]);
                }
            load_scales(k_begin + (st + 1) * kStageK);
            if (!wait_phase(c_full + 8 * cs, cp, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutFull);
            const uint32_t from = codes + cs * kTileM * 128 + row * 128;
#pragma unroll
            for (int c = 0; c < kMine; ++c) {
                if (step >= steps) break;
                step += kSets;
                while (ws >= plan.rings[1]) ws -= plan.rings[1], wp ^= 1;
                uint32_t w[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[h][0]), "=r"(w[h][1]), "=r"(w[h][2]), "=r"(w[h][3])
                                 : "r"(from + (((2 * (c * kSets + set) + h) ^ (row & 7)) << 4)));
                const uint32_t slot = to + ws * kWeightCols;
                if constexpr (TERMS) {  // sixteen weights at a time: both terms of all would not fit the registers
                    if (!wait_phase(w_empty + 8 * ws, wp ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAccFree);
                    tc_fence_after();
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        uint32_t out[8], rest[8];
                        weight_terms16<BF, EX>(w[h / 2][h % 2 * 2], w[h / 2][h % 2 * 2 + 1], hi[c][h / 2 % CH],
                                               lo[c][h / 2 % CH], z[c][h / 2 % CH], out, rest);
                        tmem_st8(slot + 8 * h, out);
                        tmem_st8(slot + 32 + 8 * h, rest);
                    }
                } else {
                    uint32_t out[4][8];
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        weights16<BF, EX>(w[h / 2][h % 2 * 2], w[h / 2][h % 2 * 2 + 1], hi[c][h / 2 % CH], lo[c][h / 2 % CH],
                                          z[c][h / 2 % CH], out[h]);
                    if (!wait_phase(w_empty + 8 * ws, wp ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAccFree);
                    tc_fence_after();
#pragma unroll
                    for (int h = 0; h < 4; ++h) tmem_st8(slot + 8 * h, out[h]);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(w_full + 8 * ws);
                ws += kSets;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(c_empty + 8 * cs);
            if (++cs == plan.rings[0]) cs = 0, cp ^= 1;
        }
        // epilogue: a warp reads its TMEM lanes; the warps of a tile's quarter share its columns, eight at a time
        if (!wait_phase(done, 0, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutAcc);
        tc_fence_after();
        const int out = o0 + row;
        const float bias = a.bias && out < n ? a.bias[out] : 0.f;
        const uint32_t acc = tmem + (TWO ? part / 2 * tile_n : 0) + (static_cast<uint32_t>(quad * 32) << 16);
        float* const partial = reinterpret_cast<float*>(smem);  // [row][output], over the rings
        // sixteen rows at a time; 16-bit results change places in shared memory (over the rings), so that a store is eight
        // outputs of a row
        uint8_t* const turned = smem + warp * (16 * 80);
        const int o_warp = o0 + row - lane;
        const bool vec = plan.y_vec && o_warp + 32 <= n;
        for (int c = (TWO ? part % 2 : part) * 16; c < tile_n; c += TWO ? 32 : 64) {
            uint32_t v[16];
            tmem_ld16_nowait(acc + c, v);
            tmem_wait();
            tmem_regs_ready(v);
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]) * back;
            if (plan.split > 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i) partial[(c + i) * kTileM + row] = f[i];
                continue;
            }
            if (a.x_scale) {
                const int r = c + lane % 16;
                const float xs = r < rows ? a.x_scale[a.x_scale_mode == kScaleRow ? r0 + r : 0] : 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) f[i] *= __shfl_sync(0xffffffffu, xs, i);
            }
            uint16_t* const y = static_cast<uint16_t*>(a.y) + (r0 + c) * a.y_stride;
            if (vec) {
                if (a.y_type == kTokF16) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        *reinterpret_cast<__half*>(turned + i * 80 + lane * 2) = __float2half_rn(f[i] + bias);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        *reinterpret_cast<__nv_bfloat16*>(turned + i * 80 + lane * 2) = __float2bfloat16_rn(f[i] + bias);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = i * 8 + lane / 4;
                    const uint4 w = *reinterpret_cast<const uint4*>(turned + r * 80 + lane % 4 * 16);
                    if (c + r < rows) *reinterpret_cast<uint4*>(y + r * a.y_stride + o_warp + lane % 4 * 8) = w;
                }
                __syncwarp();
            } else if (out < n) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (c + i < rows) tok_store16(y, i * a.y_stride + out, a.y_type, f[i] + bias);
            }
        }
        tc_fence_before();
    }
    if (plan.split > 1) {  // each block adds up a share of the rows over the cluster
        __syncwarp();
        cluster_sync();
        const uint32_t base = smem_u32(smem);
        const int mine = (rows - rank + plan.split - 1) / plan.split;  // rows rank, rank + split, ...
        for (int i = threadIdx.x; i < mine * (kTileM / 4); i += blockDim.x) {
            const int r = rank + i / (kTileM / 4) * plan.split, o = o0 + i % (kTileM / 4) * 4;
            if (o >= n) continue;
            const uint32_t at = base + (r * kTileM + i % (kTileM / 4) * 4) * 4;
            float4 v[8];
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < plan.split) v[p] = ld_cluster4(at, p);
            float f[4] = {};
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < plan.split) f[0] += v[p].x, f[1] += v[p].y, f[2] += v[p].z, f[3] += v[p].w;
            const float xs = a.x_scale ? a.x_scale[a.x_scale_mode == kScaleRow ? r0 + r : 0] : 1.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (o + e < n)
                    tok_store16(a.y, (r0 + r) * a.y_stride + o + e, a.y_type, f[e] * xs + (a.bias ? a.bias[o + e] : 0.f));
        }
        cluster_sync();
    }
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        tmem_dealloc(tmem, plan.tmem_cols);
    }
}

template <bool BF, bool TWO, bool TMA, int SS, int CH, bool EX, bool TERMS>
cudaError_t launch(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s) {
    constexpr int kTileM = TWO ? 256 : 128;
    auto* kern = w4_many_kernel<BF, TWO, TMA, SS, CH, EX, TERMS>;
    CUtensorMap codes, rows;
    cudaError_t e = tmap_rows(&codes, a.w.codes, 8, a.w.k / 16, a.w.n, a.w.k / 2, kTileM);
    if (e == cudaSuccess) {
        if (TMA)
            e = tmap_rows(&rows, a.x, 2, a.w.k, a.rows, a.x_stride * 2, p.tile_n);
        else if (p.raw_slots)
            e = tmap_rows(&rows, a.x, 8, a.w.k / 8, a.rows, a.x_stride, p.tile_n);
        else
            rows = codes;
    }
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.w.n + kTileM - 1) / kTileM * p.split, (a.rows + p.tile_n - 1) / p.tile_n);
    cfg.blockDim = dim3(TMA ? 19 * 32 : 22 * 32);
    cfg.dynamicSmemBytes = p.bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.split > 1 ? 1 : 0;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, kern, a, p, codes, rows);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

template <bool BF, bool TWO, bool TMA, int SS, bool TERMS = false>
cudaError_t launch(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s) {
    const bool exact = a.w.scale_type == (BF ? kTokBF16 : kTokF16);
    if (a.w.group % kStepK == 0)
        return exact ? launch<BF, TWO, TMA, SS, 1, true, TERMS>(a, p, s) : launch<BF, TWO, TMA, SS, 1, false, TERMS>(a, p, s);
    return exact ? launch<BF, TWO, TMA, SS, 2, true, TERMS>(a, p, s) : launch<BF, TWO, TMA, SS, 2, false, TERMS>(a, p, s);
}
template <bool BF>
cudaError_t launch_typed(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s) {
    if constexpr (BF) {
        if (p.terms && p.slot_steps == 2)
            return p.x_tma ? launch<BF, false, true, 2, true>(a, p, s) : launch<BF, false, false, 2, true>(a, p, s);
        if (p.terms) return p.x_tma ? launch<BF, false, true, 4, true>(a, p, s) : launch<BF, false, false, 4, true>(a, p, s);
    }
    if (p.two) return p.x_tma ? launch<BF, true, true, 1>(a, p, s) : launch<BF, true, false, 1>(a, p, s);
    if (p.slot_steps == 2) return p.x_tma ? launch<BF, false, true, 2>(a, p, s) : launch<BF, false, false, 2>(a, p, s);
    return p.x_tma ? launch<BF, false, true, 4>(a, p, s) : launch<BF, false, false, 4>(a, p, s);
}

}  // namespace
}  // namespace fxk
