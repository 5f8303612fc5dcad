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
    // Tiles of 128 outputs by up to 256 rows, or of 256 by 192, of the size that spreads the rows evenly. A turn of 148 of
    // the larger ones takes 1.5 times as long, or 1.1 times where warps bring the rows, which then bound it (us, smaller
    // against larger; bf16: 1536 x 4096 -> 4096 50 and 40, 1024 x 4096 -> 14336 102 and 119, 4096 rows 352 and 364; e4m3:
    // 1024 x 4096 -> 4096 49 and 49, 576 x 4096 -> 14336 109 and 107, 4096 rows 609 and 483)
    auto across = [&](int m) { return (a.w.n + m - 1) / m; };
    auto turns = [&](int m, int most) {
        return (across(m) * ((static_cast<int64_t>(a.rows) + most - 1) / most) + sms - 1) / sms;
    };
    // f16 results of bf16 rows hold more bits than a bf16 weight: a weight is two terms there, an MMA each
    p.terms = a.x_type == kTokBF16 && a.y_type == kTokF16;
    const bool two = p.two = p.terms   ? false
                             : p.x_tma ? turns(256, 192) * 3 < turns(128, 256) * 2
                                       : turns(256, 192) * 11 < turns(128, 256) * 10;
    const int tile_m = two ? 256 : 128, most_n = two ? 192 : 256;
    const int64_t tiles_n = (static_cast<int64_t>(a.rows) + most_n - 1) / most_n;
    p.tile_n = static_cast<int>((a.rows + tiles_n * 16 - 1) / (tiles_n * 16)) * 16;
    const int64_t tiles = across(tile_m) * tiles_n;
    const int all_stages = (a.w.k + kStageK - 1) / kStageK;
    // few tiles: a cluster shares one, each block a range of k, in the largest clusters that all run at once (on a GPU of
    // 148 SMs 74 of 2, 45 of 3, 33 of 4, 26 of 5, 22 of 6, 15 of 8) and leave a block two stages of codes (us without and
    // with: 16 x 4096 -> 4096 18.5 and 10.0, 256 x 4096 -> 4096 26.5 and 16.5, 192 x 8192 -> 8192 46 and 29; clusters of
    // 4, three of 36 left over for a second turn, against 3: 24 x 4096 -> 4608 18.7 and 11.9)
    int split = 1;
    for (int c = 8; !two && c > 1 && split == 1; --c) {
        if (tiles * c > sms || all_stages < 2 * c) continue;
        int most = 0;
        if (const cudaError_t e = w4_many_clusters(c, &most); e != cudaSuccess) return e;
        if (tiles <= most) split = c;
    }
    p.stages_each = (all_stages + split - 1) / split;
    p.split = (all_stages + p.stages_each - 1) / p.stages_each;  // no block without a stage
    // TMEM, all of it (a block's shared memory leaves room for no other block): accumulators, then stages of weights
    p.weight_col = (two ? 2 : 1) * p.tile_n;
    p.tmem_cols = 512;
    p.rings[1] = std::min((p.tmem_cols - p.weight_col) / (two || p.terms ? 64 : 32), kMaxRing);
    // the issuing thread's waits bound short steps: four or two of them share a slot of the rows, as room allows (4096 ->
    // 14336 bf16, us, one step a slot against more: 16 rows 23.6 and 19.5, 128 rows 25.6 and 22.3; 1024 x 4096 -> 4096
    // 28.2 and 26.9)
    p.slot_steps = two ? 1 : p.tile_n <= 128 ? 4 : 2;
    if (p.raw_slots && p.slot_steps == 4) p.raw_slots = 4;
    const int tops_bytes = 1024, w = tile_m * 128, x = p.tile_n * 128 * p.slot_steps;
    // Warps that write a slot each, taking steps in turn, tell a slot's uses apart by parity: a ring as long as they are
    // many keeps one that runs ahead from meeting a slot two uses behind.
    p.rings[0] = 2;
    p.rings[2] = !p.x_tma && p.slot_steps == 1 ? kRowWarps : 2;
    // the rest: codes and rows in turn
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
