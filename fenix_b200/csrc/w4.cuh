// w4.cuh — what the kernels of the 4-bit linear layer share.
#pragma once

#include "ptx.cuh"
#include "token.cuh"

namespace fxk {

constexpr int kStageK = 256;  // inputs of a stage of codes: 128 bytes an output
constexpr int kStepK = 64;    // inputs of a stage of operands: 128 bytes of 16-bit values a row
constexpr int kMaxRing = 8;
constexpr int kRowWarps = 4;  // that write rows which TMA does not bring
constexpr int kSmemMax = 226 * 1024;

struct ManyPlan {
    int tile_n;           // rows of a tile: a multiple of 16, at most 256
    int rings[3];         // stages of codes, weights, rows; at most kMaxRing
    int codes, rows, raw, tops;  // offsets in shared memory
    int bytes;
    int split;            // blocks of a cluster that share a tile, each with a range of k
    int stages_each;      // stages of codes of a block
    int tmem_cols;
    int weight_col;       // of the weights in TMEM, behind the accumulators: 32 columns per 128 outputs, stage and term
    int raw_slots;        // of e4m3 rows by TMA, 128 inputs each
    bool y_vec;           // results aligned to eight outputs
    int slot_steps;       // steps of 64 inputs that share a slot of the rows' ring
    bool x_tma, x_vec;    // rows come by TMA as they are; rows aligned to eight values
    bool two;             // tiles of 256 outputs
    bool terms;           // a weight is the sum of two 16-bit values
};

cudaError_t w4_many_bf16(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s);
cudaError_t w4_many_f16(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s);
// Clusters of `size` blocks that the current device runs at once.
cudaError_t w4_many_clusters(int size, int* count);
cudaError_t launch_w4_many(const W4LinearArgs& a, int sms, cudaStream_t s);
// The status word of each file's kernels, cleared.
cudaError_t w4_few_status(uint32_t* code);
cudaError_t w4_many_bf16_status(uint32_t* code);
cudaError_t w4_many_f16_status(uint32_t* code);

#ifdef __CUDACC__
// Set by a kernel of this file's includer whose bounded wait gave up; read and cleared by take_status.
static __device__ uint32_t g_w4_status;
__device__ __forceinline__ void set_w4_status(uint32_t code) { set_status(&g_w4_status, code); }

// Bounded wait for a phase. Gives up after limit_ns, or when another role of the block has. The clock is read only
// after many tries (each may sleep for a while in hardware): an ordinary wait costs no more than itself.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, const volatile int* abort, uint64_t limit_ns) {
    uint64_t t0 = 0;
    for (uint32_t it = 0;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if (it % 64 == 63) {
            if (abort && *abort) return false;
            const uint64_t now = globaltimer_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > limit_ns) return false;
        }
    }
}

// (w & mask) | bits
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}

// Eight e4m3 (in x, y) or 16-bit values at p as they lie in memory; vec: p is aligned to eight of them.
__device__ __forceinline__ uint4 raw_eight(const uint8_t* p, int x_type, bool vec) {
    uint32_t v[4] = {};
    if (x_type == kTokE4M3) {
        if (vec) {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            return make_uint4(u.x, u.y, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
            v[e] = __ldg(p + 4 * e) | __ldg(p + 4 * e + 1) << 8 | __ldg(p + 4 * e + 2) << 16 | __ldg(p + 4 * e + 3) << 24;
        return make_uint4(v[0], v[1], 0, 0);
    }
    if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
    const uint16_t* const q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __ldg(q + 2 * e) | static_cast<uint32_t>(__ldg(q + 2 * e + 1)) << 16;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// Them as 16-bit values: e4m3 widened to f16, others as they are.
__device__ __forceinline__ uint4 widened(const uint4& v, int x_type) {
    if (x_type != kTokE4M3) return v;
    const uint32_t w[2] = {v.x, v.y};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (16 * (i % 2))), __NV_E4M3);
        r[i] = reinterpret_cast<const uint32_t&>(h);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

static inline cudaError_t take_status(uint32_t* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_w4_status, sizeof *code);
    const uint32_t zero = 0;
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_w4_status, &zero, sizeof zero);
    return e;
}
#endif

}  // namespace fxk
