// w4_many.cu — how the tensor-core kernel of the 4-bit linear layer cuts a call into tiles, clusters and rings.
#include "w4.cuh"

#include <algorithm>

namespace fxk {

cudaError_t launch_w4_many(const W4LinearArgs& a, int sms, cudaStream_t s) {
    ManyPlan p{};
    const int64_t xb = a.x_type == kTokE4M3 ? 1 : 2;
    p.x_vec = reinterpret_cast<uintptr_t>(a.x) % (8 * xb) == 0 && a.x_stride % 8 == 0;
    p.x_tma = xb == 2 && p.x_vec && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
    p.y_vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_stride % 8 == 0;
    p.raw_slots = xb == 1 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 16 == 0 ? 2 : 0;
    const bool two = p.two = (a.w.n + 255) / 256 * ((a.rows + 191) / 192) >= sms;
    const int tile_m = two ? 256 : 128, most_n = two ? 192 : 256;
    p.tile_n = a.rows >= most_n ? most_n : (a.rows + 15) / 16 * 16;
    const int64_t tiles_n = (a.rows + p.tile_n - 1) / p.tile_n;
    const int64_t tiles = (a.w.n + tile_m - 1) / tile_m * tiles_n;
    const int all_stages = (a.w.k + kStageK - 1) / kStageK;
    // few tiles: a cluster shares one, each block a range of k, while a block keeps two stages of codes
    p.split = 1;
    while (!two && p.split < 8 && tiles * p.split * 2 <= sms && all_stages >= p.split * 4) p.split *= 2;
    p.stages_each = (all_stages + p.split - 1) / p.split;
    // TMEM, all of it (a block's shared memory leaves room for no other block): accumulators, then stages of weights
    p.weight_col = (two ? 2 : 1) * p.tile_n;
    p.tmem_cols = 512;
    p.rings[1] = std::min((p.tmem_cols - p.weight_col) / (two ? 64 : 32), kMaxRing);
    // shared memory: codes and rows in turn
    // short steps: four to a slot, for fewer waits
    p.slot_steps = !two && p.tile_n <= 64 ? 4 : 1;
    if (p.raw_slots && p.slot_steps == 4) p.raw_slots = 4;
    const int tops_bytes = 1024, w = tile_m * 128, x = p.tile_n * 128 * p.slot_steps;
    // Warps that write a slot each, taking steps in turn, tell a slot's uses apart by parity: a ring as long as they are
    // many keeps one that runs ahead from meeting a slot two uses behind.
    p.rings[0] = 2;
    p.rings[2] = !p.x_tma && p.slot_steps == 1 ? kRowWarps : 2;
    int room = kSmemMax - tops_bytes - p.rings[0] * w - p.rings[2] * x - p.raw_slots * p.tile_n * 128;
    if (room < 0) return cudaErrorInvalidConfiguration;
    for (bool more = true; more;) {
        more = false;
        for (int i : {2, 0}) {
            const int cost = i == 2 ? x : w;
            if (p.rings[i] < kMaxRing && room >= cost) {
                ++p.rings[i];
                room -= cost;
                more = true;
            }
        }
    }
    p.codes = 0;
    p.rows = p.rings[0] * w;
    p.raw = p.rows + p.rings[2] * x;
    p.tops = p.raw + p.raw_slots * p.tile_n * 128;
    p.bytes = p.tops + tops_bytes;
    if (p.split > 1) {  // the partial sums lie over the rings
        const int partial = p.tile_n * tile_m * 4;
        if (partial > p.tops) {
            p.tops = partial;
            p.bytes = partial + tops_bytes;
        }
    }
    return a.x_type == kTokBF16 ? w4_many_bf16(a, p, s) : w4_many_f16(a, p, s);
}

}  // namespace fxk
