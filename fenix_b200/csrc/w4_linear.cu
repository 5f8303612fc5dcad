// w4_linear.cu — linear layer with 4-bit weights and group scales.
#include "counters.hpp"
#include "ptx.cuh"
#include "tmap.hpp"
#include "token.cuh"
#include "w4.cuh"

#include <algorithm>

namespace fxk {
namespace {

// ---- few rows ----------------------------------------------------------------------------------
// With up to 8 token rows the floor is the weights' way from memory: 4.1 bits a weight, each used once per row. What
// bounds the kernel before that is the instructions that make operands of the codes and the time a warp's chain of
// them takes (1 x 8192 -> 28672 f16: 32 us, 3.7 TB/s, 57% of the copy's rate; 1 x 4096 -> 4096: 6.5 us, of which half
// is launch, first loads and the reduction; 8 x 4096 -> 14336 e4m3 with zero points: 18.5 us). One block per SM walks
// over tiles of 32 outputs (the last of them over tiles of 16, so that all blocks have as much to do): a producer warp
// keeps a ring of TMA boxes, 32 outputs x 256 inputs, ahead of the consumer warps, across tiles, so that memory never
// waits for a tile's end (a bulk copy for each row of a tile costs its thread some 60 ns); each consumer takes 128
// inputs of a stage. Codes meet the rows in m16n8k16 MMAs (A: outputs x inputs, B: inputs x 8 rows), whose 8 columns are
// what few rows can fill: a tcgen05 operand would have to be written before it is read (all of it: 1 x 4096 -> 4096
// 9.5 us, 1 x 8192 -> 28672 f16 57). The rows lie in shared memory for the whole walk, converted once and in the MMA's order.
// A weight enters the MMA as code - zero, a whole number (in bf16 times 2^-11), made of two codes at a time by one
// logical operation and one packed subtraction, both exact. So every product is exact, the sums hold nothing but the
// result's own terms, and scales are applied in f32 to the sum of a group's inputs: no weight is rounded. The consumers'
// partial sums meet in shared memory.

constexpr int kBlockK = 128;  // inputs of a consumer warp in a stage
// (us, with 16, 18 and 22: 1 x 8192 -> 28672 f16 32.3, 33.6 and 33.0, 8 x 8192 -> 8192 22.8, 23.4 and 32.7)
constexpr int kMaxConsumers = 16;

template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if (BF)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Nibbles (i, i + 4) of a word of eight codes as two 16-bit floats code - zero, by or'ing them into the mantissa of a
// power of two and taking off that and the zero point. f16: 1024 + code, whose last place is one, or 64 + code, whose
// last place is a sixteenth, wherever the nibble lies (one shift for a word's four pairs). bf16: (128 + code) 2^-11
// (three shifts); the factor keeps the sum of 128 inputs of any size, times up to 15 each, inside f32's range.
template <bool BF>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, const uint32_t (&offset)[2]) {
    const uint32_t v = BF ? and_or(w >> (4 * i), 0x000f000fu, 0x3d803d80u)
                          : and_or(i >= 2 ? w >> 8 : w, i & 1 ? 0x00f000f0u : 0x000f000fu, i & 1 ? 0x54005400u : 0x64006400u);
    uint32_t r;
    if (BF)
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(offset[0]));
    else
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(offset[i & 1]));
    return r;
}
// What code_pair takes off for a zero point, for even and odd i.
template <bool BF>
__device__ __forceinline__ void code_offsets(uint32_t zero, uint32_t (&offset)[2]) {
    offset[0] = (BF ? 0x3d803d80u : 0x64006400u) + 0x00010001u * zero;
    offset[1] = 0x54005400u + 0x00100010u * zero;
}
constexpr float kBackBF16 = 2048.f;  // bf16's factor leaves with the scales' sum

// Eight 16-bit values as the pairs (i, i + 4), i = 0..3: code_pair's order.
__device__ __forceinline__ uint4 paired(const uint4& v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
}

// How the few-rows kernel walks and where its parts lie in shared memory; made by the host.
struct FewPlan {
    int consumers;   // warps, even; a stage is 128 inputs for each
    int stages;      // of the ring
    int seg_blocks;  // blocks of 128 inputs whose rows and scales are in shared memory at once, a multiple of consumers
    int wide;        // tiles of 32 outputs, all blocks having as many; the outputs after them go in tiles of 16
    int tiles;
    int x_pitch;     // of a row's inputs: 64 modulo 128, so that 2 rows x 4 lanes of 16 bytes hit all banks once
    int s_pitch, z_pitch;  // of an output's scales and zero points: 16 modulo 128, so that 8 outputs hit different banks
    int red_bufs;  // tiles whose partial sums have room
    int x, scale, accum, red, ring, bytes;  // offsets; accum: the sums of earlier segments, by tile of this block
    bool x_vec;
};

constexpr int kM = 32;  // outputs of a wide tile
constexpr int kMaxStages = 6;

__device__ __forceinline__ void consumers_sync(int warps) { asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory"); }

// Bytes [0, bytes) of each of `rows` rows, `src_pitch` apart, to shared memory rows `dst_pitch` apart by one warp:
// asynchronously in pieces of UNIT bytes where the addresses allow it, else by plain stores, byte by byte (the result:
// whether asynchronously).
template <int UNIT>
__device__ __forceinline__ void rows_async(uint32_t dst, int dst_pitch, const uint8_t* src, int64_t src_pitch, int rows,
                                           int bytes) {
    const int lane = threadIdx.x % 32;
    for (int r = lane / 4; r < rows; r += 8)
        for (int at = lane % 4 * UNIT; at < bytes; at += 4 * UNIT) {
            const uint32_t to = dst + r * dst_pitch + at;
            const uint8_t* const from = src + r * src_pitch + at;
            if constexpr (UNIT == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
        }
}
__device__ __forceinline__ bool rows_to_shared(uint8_t* to, int dst_pitch, const uint8_t* src, int64_t src_pitch, int rows,
                                               int bytes) {
    const int64_t all = static_cast<int64_t>(reinterpret_cast<uintptr_t>(src)) | src_pitch;
    if (all % 16 == 0 && bytes % 16 == 0) {
        rows_async<16>(smem_u32(to), dst_pitch, src, src_pitch, rows, bytes);
        return true;
    } else if (all % 4 == 0 && bytes % 4 == 0) {
        rows_async<4>(smem_u32(to), dst_pitch, src, src_pitch, rows, bytes);
        return true;
    }
    const int lane = threadIdx.x % 32;
    for (int r = lane / 4; r < rows; r += 8)
#pragma unroll 8
        for (int at = lane % 4; at < bytes; at += 4) to[r * dst_pitch + at] = __ldg(src + r * src_pitch + at);
    return false;
}

// CPF chunks of 32 inputs times MT m-tiles of 16 outputs into acc, under one scale per output. The codes of output
// m 16 + h 8 (+ this lane's g, in `codes`) lie 128 bytes apart, 16-byte cell c of them at cell c ^ g (cell: of the first
// chunk); x_at: this lane's row; scales and zero points as they are stored.
template <bool BF, int CPF, bool Z, int MT>
__device__ __forceinline__ void unit(float (&acc)[2][4], uint32_t codes, uint32_t x_at, int cell, uint32_t s_at, int s_pitch,
                                     int scale_type, uint32_t z_at, int z_pitch) {
    uint32_t x[CPF][4], w[MT][2][CPF], offset[MT][2][2];
    float scale[MT][2], part[MT][4] = {};
#pragma unroll
    for (int c = 0; c < CPF; ++c) {
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[c][0]), "=r"(x[c][1]), "=r"(x[c][2]), "=r"(x[c][3])
                     : "r"(x_at + c * 64));
        const uint32_t at = codes + (cell ^ c) * 16;  // the first chunk's cell is a multiple of CPF before the swizzle
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[m][h][c]) : "r"(at + (m * 16 + h * 8) * 128));
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = s_at + (m * 16 + h * 8) * s_pitch;
            if (scale_type == kTokF32) {
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(scale[m][h]) : "r"(at));
            } else {
                unsigned short raw;
                asm volatile("ld.shared.b16 %0, [%1];" : "=h"(raw) : "r"(at));
                scale[m][h] = scale_type == kTokF16 ? __half2float(__ushort_as_half(raw))
                                                    : __uint_as_float(static_cast<uint32_t>(raw) << 16);
            }
            uint32_t zero = 8;
            if (Z) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(zero) : "r"(z_at + (m * 16 + h * 8) * z_pitch));
            code_offsets<BF>(zero, offset[m][h]);
        }
#pragma unroll
    for (int c = 0; c < CPF; ++c)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
                mma16816<BF>(part[m], code_pair<BF>(w[m][0][c], i, offset[m][0]), code_pair<BF>(w[m][1][c], i, offset[m][1]),
                             code_pair<BF>(w[m][0][c], i + 1, offset[m][0]), code_pair<BF>(w[m][1][c], i + 1, offset[m][1]),
                             x[c][i], x[c][i + 1]);
        }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][e] = fmaf(scale[m][e / 2], part[m][e], acc[m][e]);
}

// CPF: the scale changes every CPF chunks of 32 inputs at most (4: groups are multiples of 128, 2: of 64, 1: of 32);
// such a unit is summed in the MMAs before its scale is applied. Lane t of a quad takes inputs 8 t .. 8 t + 7 of a
// chunk, as code words and rows lie. Besides the consumers: a warp that issues the codes' TMA loads, 128 bytes x 16
// outputs each, and one that brings a tile's scales (and zero points: Z) to shared memory a tile ahead.
template <bool BF, int CPF, bool Z>
__global__ void __launch_bounds__((kMaxConsumers + 2) * 32, 1)
    w4_few_kernel(const __grid_constant__ W4LinearArgs a, const __grid_constant__ FewPlan plan,
                  const __grid_constant__ CUtensorMap map_wide, const __grid_constant__ CUtensorMap map_narrow) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 4];  // ring full, ring empty, scales full, scales empty
    __shared__ volatile int abort_flag;
    constexpr int kUnits = 4 / CPF;
    const int warps = plan.consumers, warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n = a.w.n, k = a.w.k, group = a.w.group;
    const int blocks = (k + kBlockK - 1) / kBlockK;
    const int rows = a.rows;  // at most 8
    const int stage_bytes = warps / 2 * kM * 128, s_bytes = kM * (plan.s_pitch + (Z ? plan.z_pitch : 0));
    const uint32_t ring = smem_u32(smem + plan.ring), full = smem_u32(bars), empty = full + 8 * kMaxStages;
    const uint32_t s_full = full + 16 * kMaxStages, s_empty = s_full + 16;
    auto tile_row = [&](int tile) { return tile < plan.wide ? tile * kM : plan.wide * kM + (tile - plan.wide) * 16; };
    auto gave_up = [&](uint32_t code) {
        abort_flag = 1;
        set_w4_status(code);
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < plan.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, warps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 32);
            mbar_init(s_empty + 8 * i, warps);
        }
        abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    int slot = 0, s_slot = 0;
    uint32_t phase = 0, s_phase = 0;

    if (warp == warps) {  // codes
        if (lane) return;
        int issued = 0;
        for (int seg = 0; seg < blocks && !a.hold_codes; seg += plan.seg_blocks) {
            const int seg_end = min(seg + plan.seg_blocks, blocks);
            for (int tile = blockIdx.x; tile < plan.tiles; tile += gridDim.x) {
                const bool wide = tile < plan.wide;
                const CUtensorMap* const map = wide ? &map_wide : &map_narrow;
                const int o0 = tile_row(tile), box_bytes = (wide ? kM : 16) * 128;
                for (int blk = seg; blk < seg_end; blk += warps) {
                    const int boxes = (min(warps, seg_end - blk) + 1) / 2;  // of 256 inputs; past the end they read as zeros
                    if (!wait_phase(empty + 8 * slot, phase ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                    if (abort_flag) break;
                    mbar_arrive_expect_tx(full + 8 * slot, boxes * box_bytes);
                    for (int i = 0; i < boxes; ++i)
                        tma_load_2d(ring + slot * stage_bytes + i * kM * 128, map, (blk / 2 + i) * 16, o0, full + 8 * slot);
                    ++issued;
                    if (++slot == plan.stages) slot = 0, phase ^= 1;
                }
            }
        }
        // consumers that give up, now or later, no longer wait for the copies still on their way
        for (int i = min(issued, plan.stages); i > 0; --i) {
            if (slot-- == 0) slot = plan.stages - 1, phase ^= 1;
            wait_phase(full + 8 * slot, phase, nullptr, a.wait_ns);
        }
        return;
    }
    const int sb = a.w.scale_type == kTokF32 ? 4 : 2;
    if (warp == warps + 1) {  // scales, as they are stored
        const int groups = k / group;
        for (int seg = 0; seg < blocks; seg += plan.seg_blocks) {
            const int seg_end = min(seg + plan.seg_blocks, blocks);
            const int g0 = seg * kBlockK / group, gn = (min(seg_end * kBlockK, k) - 1) / group + 1 - g0;
            for (int tile = blockIdx.x; tile < plan.tiles; tile += gridDim.x) {
                if (!wait_phase(s_empty + 8 * s_slot, s_phase ^ 1, &abort_flag, a.wait_ns)) gave_up(kStatusTimeoutEmpty);
                uint8_t* const to = smem + plan.scale + s_slot * s_bytes;
                const int o0 = tile_row(tile), per = min(tile < plan.wide ? kM : 16, n - o0);
                const int64_t at = static_cast<int64_t>(o0) * groups + g0;
                bool async = rows_to_shared(to, plan.s_pitch, static_cast<const uint8_t*>(a.w.scales) + at * sb,
                                            static_cast<int64_t>(groups) * sb, per, gn * sb);
                if (Z) async &= rows_to_shared(to + kM * plan.s_pitch, plan.z_pitch, a.w.zeros + at, groups, per, gn);
                if (async) {
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(s_full + 8 * s_slot) : "memory");
                } else {  // an arrival of this thread's own, which releases its plain stores, too
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    mbar_arrive(s_full + 8 * s_slot);
                }
                if (++s_slot == 2) s_slot = 0, s_phase ^= 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }

    // (rows past the last: nothing reads their sums)
    const uint32_t x_lane = smem_u32(smem + plan.x) + min(g, rows - 1) * plan.x_pitch + t * 16;
    const float inv_group = 1.f / static_cast<float>(group);
    for (int seg = 0; seg < blocks; seg += plan.seg_blocks) {
        const int seg_end = min(seg + plan.seg_blocks, blocks), g0 = seg * kBlockK / group;
        if (seg) consumers_sync(warps);  // the last segment's rows are read
        {  // the rows' inputs of this segment
            const int kxb = a.x_type == kTokE4M3 ? 1 : 2, eights = min((seg_end - seg) * kBlockK, k - seg * kBlockK) / 8;
            for (int r = 0; r < rows; ++r) {
                const uint8_t* const p = static_cast<const uint8_t*>(a.x) + (r * a.x_stride + seg * kBlockK) * kxb;
                for (int i = warp * 32 + lane; i < eights; i += warps * 32)
                    *reinterpret_cast<uint4*>(smem + plan.x + r * plan.x_pitch + i * 16) =
                        paired(widened(raw_eight(p + i * 8 * kxb, a.x_type, plan.x_vec), a.x_type));
            }
        }
        consumers_sync(warps);
        int turn = 0, added = 0;  // tiles of this block, and those added up
        for (int tile = blockIdx.x; tile < plan.tiles; tile += gridDim.x, ++turn) {
            const bool wide = tile < plan.wide;
            float acc[2][4] = {};
            if (!wait_phase(s_full + 8 * s_slot, s_phase, &abort_flag, a.wait_ns))
                gave_up(kStatusTimeoutFull);
            const uint32_t s_at = smem_u32(smem + plan.scale + s_slot * s_bytes) + g * plan.s_pitch;
            const uint32_t z_at = smem_u32(smem + plan.scale + s_slot * s_bytes) + kM * plan.s_pitch + g * plan.z_pitch;
            for (int blk0 = seg; blk0 < seg_end; blk0 += warps) {
                const int blk = blk0 + warp, k0 = blk * kBlockK;
                if (!wait_phase(full + 8 * slot, phase, &abort_flag, a.wait_ns))
                    gave_up(kStatusTimeoutFull);
                if (blk < seg_end) {
                    const uint32_t cw = ring + slot * stage_bytes + warp / 2 * kM * 128 + g * 128 + t * 4;
                    const uint32_t xw = x_lane + (k0 - seg * kBlockK) * 2;
#pragma unroll
                    for (int u = 0; u < kUnits; ++u) {
                        const int kc = k0 + u * 32 * CPF;
                        if (CPF < 4 && kc >= k) break;
                        // (kc + 1/2) / group truncated: exact while k < 2^21
                        const int gi =
                            (k < (1 << 21) ? static_cast<int>((static_cast<float>(kc) + 0.5f) * inv_group) : kc / group) - g0;
                        const int cell = (4 * (warp & 1) + u * CPF) ^ g;
                        if (wide)
                            unit<BF, CPF, Z, 2>(acc, cw, xw + u * CPF * 64, cell, s_at + gi * sb, plan.s_pitch, a.w.scale_type,
                                                z_at + gi, plan.z_pitch);
                        else
                            unit<BF, CPF, Z, 1>(acc, cw, xw + u * CPF * 64, cell, s_at + gi * sb, plan.s_pitch, a.w.scale_type,
                                                z_at + gi, plan.z_pitch);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + 8 * slot);
                if (++slot == plan.stages) slot = 0, phase ^= 1;
            }
            if (lane == 0) mbar_arrive(s_empty + 8 * s_slot);
            if (++s_slot == 2) s_slot = 0, s_phase ^= 1;
            // partial sums [tile][warp][row][output]: warps go on to the next tile, and add up when the buffers are full
            const int per_tile = rows * kM;
            float* const red = reinterpret_cast<float*>(smem + plan.red) + (turn - added) * warps * per_tile;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 2 * t + (e & 1);
                    if (r < rows) red[warp * per_tile + r * kM + m * 16 + (e / 2) * 8 + g] = acc[m][e];
                }
            const bool last = tile + static_cast<int>(gridDim.x) >= plan.tiles;
            if (turn + 1 - added < plan.red_bufs && !last) continue;
            consumers_sync(warps);
            for (int i = threadIdx.x; i < (turn + 1 - added) * per_tile; i += warps * 32) {
                const int nth = i / per_tile, r = i % per_tile / kM;
                const int from = tile - (turn - added - nth) * static_cast<int>(gridDim.x);
                const int o = tile_row(from) + i % kM;
                if (i % kM >= (from < plan.wide ? kM : 16) || o >= n) continue;
                const float* const part = reinterpret_cast<float*>(smem + plan.red) + nth * warps * per_tile + i % per_tile;
                float v = 0.f, v1 = 0.f;
#pragma unroll 4
                for (int w = 0; w < warps; w += 2) {
                    v += part[w * per_tile];
                    v1 += part[(w + 1) * per_tile];
                }
                v += v1;
                float* const kept = reinterpret_cast<float*>(smem + plan.accum) + added * per_tile + i;
                if (seg) v += *kept;
                if (seg_end < blocks) {
                    *kept = v;
                } else {
                    if (BF) v *= kBackBF16;
                    if (a.x_scale) v *= a.x_scale[a.x_scale_mode == kScaleRow ? r : 0];
                    if (a.bias) v += a.bias[o];
                    tok_store16(a.y, r * a.y_stride + o, a.y_type, v);
                }
            }
            added = turn + 1;
            if (!last) consumers_sync(warps);
        }
    }
}

constexpr int kFewSmem = 226 * 1024;  // a block's shared memory, less the barriers

int round_up(int v, int to) { return (v + to - 1) / to * to; }

FewPlan few_plan(const W4LinearArgs& a, int rows, int sms, int* grid) {
    constexpr int kXRoom = 80 * 1024, kScaleRoom = 24 * 1024;  // for the rows, and one tile's scales, at most
    FewPlan p{};
    const int blocks = (a.w.k + kBlockK - 1) / kBlockK;
    // as many consumers as leave the fewest idle in a tile's last stage
    const int turns = (blocks + kMaxConsumers - 1) / kMaxConsumers;
    p.consumers = round_up((blocks + turns - 1) / turns, 2);
    const int x_fit = kXRoom / rows / (p.consumers * kBlockK * 2 + 64);
    const int sb = a.w.scale_type == kTokF32 ? 4 : 2;
    const int64_t s_room = (kScaleRoom / kM - 2 * 128) / (a.w.zeros ? sb + 1 : sb) - 1;
    const int64_t s_fit = s_room * a.w.group / (p.consumers * kBlockK);
    int fit = x_fit < s_fit ? x_fit : static_cast<int>(s_fit);
    if (fit < 1) fit = 1;
    const int segs = (turns + fit - 1) / fit;
    p.seg_blocks = (turns + segs - 1) / segs * p.consumers;
    p.x_pitch = round_up(p.seg_blocks * kBlockK * 2, 128) + 64;
    const int seg_k = p.seg_blocks < blocks ? p.seg_blocks * kBlockK : a.w.k;
    const int seg_groups = (seg_k + a.w.group - 1) / a.w.group + 1;  // a segment may begin inside a group
    p.s_pitch = round_up(seg_groups * sb, 128) + 16;
    p.z_pitch = round_up(seg_groups, 128) + 16;
    *grid = sms;
    p.wide = a.w.n / kM / sms * sms;
    p.tiles = p.wide + (a.w.n - p.wide * kM + 15) / 16;
    if (p.tiles < sms) *grid = p.tiles;
    p.x = 0;
    p.scale = round_up(rows * p.x_pitch, 128);
    p.accum = p.scale + round_up(2 * kM * (p.s_pitch + (a.w.zeros ? p.z_pitch : 0)), 128);
    p.red = p.accum;
    if (p.seg_blocks < blocks) {  // room for the sums of a block's tiles between segments
        const int per = 16 * 1024 / (rows * kM * 4);
        if ((p.tiles + *grid - 1) / *grid > per) *grid = (p.tiles + per - 1) / per;
        p.red += round_up((p.tiles + *grid - 1) / *grid * rows * kM * 4, 128);
    }
    // partial sums of as many tiles as have room beside three stages: a warp need not wait for the others at a tile's end
    // (1 x 8192 -> 28672 f16 32.3 us, 35.4 with two buffers; 8 x 8192 -> 8192 22.8 us with three, 25.0 with one)
    const int stage = p.consumers / 2 * kM * 128, per_tile = p.consumers * rows * kM * 4;
    p.red_bufs = std::clamp(48 * 1024 / per_tile, 1, (p.tiles + *grid - 1) / *grid);
    auto place = [&] {
        p.ring = round_up(p.red + p.red_bufs * per_tile, 1024);
        p.stages = std::min((kFewSmem - p.ring) / stage, kMaxStages);
        return p.stages >= 3 || p.red_bufs == 1;
    };
    while (!place()) --p.red_bufs;
    p.bytes = p.ring + p.stages * stage;
    return p;
}

template <bool BF, int CPF, bool Z>
cudaError_t launch_few(const W4LinearArgs& a, bool x_vec, cudaStream_t s) {
    auto* kern = w4_few_kernel<BF, CPF, Z>;
    int grid;
    FewPlan p = few_plan(a, a.rows, sm_count(), &grid);
    p.x_vec = x_vec;
    CUtensorMap wide, narrow;
    cudaError_t e = tmap_rows(&wide, a.w.codes, 8, a.w.k / 16, a.w.n, a.w.k / 2, kM);
    if (e == cudaSuccess) e = tmap_rows(&narrow, a.w.codes, 8, a.w.k / 16, a.w.n, a.w.k / 2, 16);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
    if (e != cudaSuccess) return e;
    count_launch();
    kern<<<grid, (p.consumers + 2) * 32, p.bytes, s>>>(a, p, wide, narrow);
    return cudaGetLastError();
}
template <bool BF, bool Z>
cudaError_t launch_few_cpf(const W4LinearArgs& a, bool x_vec, cudaStream_t s) {
    if (a.w.group % 128 == 0) return launch_few<BF, 4, Z>(a, x_vec, s);
    if (a.w.group % 64 == 0) return launch_few<BF, 2, Z>(a, x_vec, s);
    return launch_few<BF, 1, Z>(a, x_vec, s);
}
cudaError_t launch_few_typed(const W4LinearArgs& a, bool x_vec, cudaStream_t s) {
    if (a.x_type == kTokBF16)
        return a.w.zeros ? launch_few_cpf<true, true>(a, x_vec, s) : launch_few_cpf<true, false>(a, x_vec, s);
    return a.w.zeros ? launch_few_cpf<false, true>(a, x_vec, s) : launch_few_cpf<false, false>(a, x_vec, s);
}

}  // namespace

cudaError_t launch_w4_linear(const W4LinearArgs& a, cudaStream_t s) {
    // 8 rows are an MMA's columns; the kernels meet there (us, few rows' and many rows': 4 x 4096 -> 14336 14.8 and 20.0,
    // 8 x 4096 -> 4096 9.1 and 9.9, 8 x 4096 -> 14336 17.3 and 20.0, 8 x 8192 -> 8192 22.8 and 21.4, 8 x 8192 -> 28672 50
    // and 60)
    if (a.rows > 8) {
        constexpr int kMost = 65535 * 16;  // rows of a launch: 65535 of the smallest tiles
        for (int64_t row0 = 0; row0 < a.rows; row0 += kMost) {
            W4LinearArgs b = a;
            b.x = static_cast<const uint8_t*>(a.x) + row0 * a.x_stride * (a.x_type == kTokE4M3 ? 1 : 2);
            b.y = static_cast<uint8_t*>(a.y) + row0 * a.y_stride * 2;
            if (a.x_scale_mode == kScaleRow) b.x_scale = a.x_scale + row0;
            b.rows = static_cast<int>(a.rows - row0 < kMost ? a.rows - row0 : kMost);
            const cudaError_t e = launch_w4_many(b, sm_count(), s);
            if (e != cudaSuccess) return e;
        }
        return cudaSuccess;
    }
    const int64_t xb = a.x_type == kTokE4M3 ? 1 : 2;
    const bool x_vec = reinterpret_cast<uintptr_t>(a.x) % (8 * xb) == 0 && a.x_stride % 8 == 0;
    return launch_few_typed(a, x_vec, s);
}

cudaError_t w4_few_status(uint32_t* code) { return take_status(code); }

}  // namespace fxk
