// kv4_rule.h — which kernel an attention call over the paged 4-bit cache takes. Host
// arithmetic alone: the tests ask it (a hook of theirs) that their sizes still reach the kernel
// they were made for.
#pragma once

namespace emb {

enum { KV4_FEW_4 = 1, KV4_FEW_8, KV4_MANY_1, KV4_MANY_2 };   // rows (row tiles) of a CTA
enum { KV4_TILE_ROWS = 128 };

// Few rows are taken eight at a time, the cache cut into pieces and read once for each
// eight: 0.045 ns for eight rows and a position (heads of 128; 0.030 of 64, 0.020 of 32). Many
// are taken 128 at a time by CTAs that go through the cache alone: 32 ns a position in fp32, 28 in
// fp16 (64: 18 and 16, 32: 15 and 13), as long as there are no more than 128 of them. The smaller
// estimate decides; the quotients are 692, 615, 619, 531, 727, 650, one number a type is near enough.
// Us, eight at a time / 128 at a time, fp32, 16 / 8 heads of 128: 1 sequence of 20,000 positions, 128 rows
// 238 / 638, 256 rows 462 / 639; 8 sequences of 1000, 32 rows 39 / 48, 64 rows 70 / 50; 64
// sequences of 1000, 8 rows 72 / 129, 32 rows 238 / 144. 14 / 2 of 64: 1 of 20,000, 256 rows 268 /
// 375; 8 / 1 of 32: 105 / 298.
//
// Of many, two row tiles go to a CTA once there are enough pairs, if a pair is more than one tile (64
// sequences of 1000, 32 rows: 144 / 174). Us, one / two:
//   heads of 128   fp32  64 pairs 64 / 68, 96 59 / 60, 128 77 / 72, 250 666 / 454
//                  fp16  32 pairs 68 / 65, 64 53 / 49, 96 49 / 44, 250 509 / 310
//   of 64          fp32  112 pairs 48 / 51, 141 217 / 225, 192 53 / 49, 440 233 / 214
//                  fp16  56 pairs 31 / 41, 112 38 / 41, 192 44 / 43, 440 180 / 173
//   of 32          fp32  64 pairs 31 / 40, 125 181 / 186, 250 111 / 101, 504 116 / 114
//                  fp16  64 pairs 26 / 35, 250 89 / 91, 504 94 / 100, 576 108 / 115: never
//
// The host knows the longest sequence's rows and the batch's: groups of rows are no more than either
// allows. 64 sequences of 2000 positions, one with 256 rows and the others with one: 147 us in the
// kernel for few, 248 in the one for many, which the longest alone would choose; 512 of 1000, one
// with 512: 908 / 1108. The kernel for few has a CTA for every eight rows that any sequence could have: too
// many that are empty cost more (201 sequences of 2000, one with 2000 rows, 134 times the groups: 1510 /
// 963), and a grid has its limits.
static inline long long kv4_groups(int size, int n_tokens, int max_q, int group, int n_kv, int n_seqs) {
    const long long each = ((long long)max_q * group + size - 1) / size * n_seqs;
    const long long all = (long long)n_tokens * group / size + n_seqs;
    return (each < all ? each : all) * n_kv;
}
static inline int kv4_kernel(int elem_bytes, int head_dim, int n_tokens, int max_q, int group, int n_kv, int n_seqs) {
    const bool f32 = elem_bytes == 4;
    const long long rows = (long long)max_q * group;
    const long long eights = kv4_groups(8, n_tokens, max_q, group, n_kv, n_seqs);
    const long long tiles = kv4_groups(KV4_TILE_ROWS, n_tokens, max_q, group, n_kv, n_seqs);
    const long long chunks = (rows + 7) / 8 * n_kv, ctas = chunks * n_seqs;
    if (eights <= (f32 ? 640 : 560) * (tiles > 128 ? tiles : 128) / 128 && ctas <= 100 * eights && chunks <= 65535 &&
        ctas <= 0x7FFFFFFF)
        return rows <= 4 ? KV4_FEW_4 : KV4_FEW_8;
    const long long pairs = kv4_groups(2 * KV4_TILE_ROWS, n_tokens, max_q, group, n_kv, n_seqs);
    if (rows <= KV4_TILE_ROWS || (head_dim == 32 && !f32)) return KV4_MANY_1;
    return pairs >= (head_dim == 128 ? (f32 ? 96 : 32) : head_dim == 64 ? (f32 ? 160 : 192) : 200) ? KV4_MANY_2 : KV4_MANY_1;
}

}  // namespace emb
