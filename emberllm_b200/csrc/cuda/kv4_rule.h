// kv4_rule.h — which kernel an attention call over the paged 4-bit cache takes. Host
// arithmetic alone: the tests ask it (a hook of theirs) that their sizes still reach the kernel
// they were made for.
#pragma once

namespace emb {

enum { KV4_FEW_4 = 1, KV4_FEW_8, KV4_MANY_1, KV4_MANY_2 };   // rows (row tiles) of a CTA
enum { KV4_TILE_ROWS = 128 };

// Few rows are taken eight at a time, the cache cut into pieces and read once for each
// eight: 0.055 ns for eight rows and a position. Many are taken 128 at a time by CTAs that
// go through the cache alone: 28 ns a position, as long as there are no more than 128 of
// them. The smaller estimate decides. Measured, eight at a time / 128 at a time, in us,
// 16 / 8 heads of 128, fp32: 1 sequence of 20,000 positions, 8 rows 16 / 544, 128 rows 125 / 548;
// 8 sequences of 1000, 64 rows 34 / 38, 128 rows 65 / 40; 64 sequences of 1000, 16 rows 67 / 148,
// 64 rows 231 / 164.
//
// Of many, two row tiles go to a CTA once there are enough of them. Us, one / two (16 / 8 heads of
// 128):
//   32 pairs (512 rows of 2000)      fp32 67 / 80     fp16 61 / 52
//   128 pairs (4 x 512 of 1200)      fp32 65 / 59     fp16 54 / 40
//   250 pairs (4000 of 8000)         fp32 605 / 403   fp16 494 / 252
static inline int kv4_kernel(int elem_bytes, int max_q, int group, int n_kv, int n_seqs) {
    const long long rows = (long long)max_q * group, heads = (long long)n_seqs * n_kv;
    const long long eights = (rows + 7) / 8 * heads, tiles = (rows + KV4_TILE_ROWS - 1) / KV4_TILE_ROWS * heads;
    if (eights <= 512 * (tiles > 128 ? tiles : 128) / 128) return rows <= 4 ? KV4_FEW_4 : KV4_FEW_8;
    const long long pairs = (rows + 2 * KV4_TILE_ROWS - 1) / (2 * KV4_TILE_ROWS) * heads;
    return pairs >= (elem_bytes == 4 ? 96 : 32) ? KV4_MANY_2 : KV4_MANY_1;
}

}  // namespace emb
