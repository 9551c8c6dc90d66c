// kv4.cuh — layout of the paged 4-bit KV cache and the batch's index arithmetic,
// shared by the kernels that write it (kv4.cu) and read it (kv4.cu, kv4_attn.cuh).
//
// One page of one kv head is one contiguous chunk of page_size / 16 groups; a group
// holds 16 positions, whole, so that one contiguous copy brings what a warp works on
// (hd = head_dim, nb = hd/32 blocks, p = position inside the group):
//
//     [16][hd/2] key codes | [8][hd] value codes | [16][nb] fp16 key scales
//     | [8][nb][2] fp16 value scales                       (18 * hd bytes)
//
// The order of the codes serves the matrix fragments that the attention builds
// from them in registers:
//   keys    row p of hd/2 bytes: word (t, b), t = 0..3, at byte t*(4*nb) + 4*b holds
//           dims b*32 + 8*t + n in nibble n: lane t of a fragment loads its words of
//           every block at once
//   values  pairs of positions share rows of hd bytes: word (g, b), g = 0..7, at
//           byte g*(4*nb) + 4*b holds dims b*32 + 4*g + n in nibble n of its lower
//           half for the even position and of its upper half for the odd one, so
//           that a masked word is a pair of operands; their scales likewise
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "ember_kv4.h"

namespace emb {

struct Kv4View {
    uint8_t *data;
    int n_pages, page_shift, n_kv;
    uint32_t chunk;               // bytes of one page of one kv head
};

struct Kv4Rows {                  // EmberKv4Batch on the device side
    const int32_t *q_start, *kv_len, *table;
    int n_seqs, table_stride, n_tokens;
    int cap;                      // table_stride * page_size, within int
};

__host__ __device__ constexpr uint32_t kv4_group(int hd) { return 18u * hd; }   // bytes of 16 positions
__host__ __device__ inline uint32_t kv4_chunk(int page_size, int hd) { return page_size / 16 * kv4_group(hd); }

// one sequence's rows and length, every number within the bounds the host knows
struct Kv4Seq {
    int row0, rows, len;          // first row, number of rows, positions in the cache
};
EMB_DEV Kv4Seq kv4_seq(const Kv4Rows &b, int i) {
    Kv4Seq s;
    int r0 = i, r1 = i + 1;
    if (b.q_start) { r0 = b.q_start[i]; r1 = b.q_start[i + 1]; }
    r0 = max(0, min(r0, b.n_tokens));
    r1 = max(r0, min(r1, b.n_tokens));
    s.row0 = r0;
    s.rows = r1 - r0;
    s.len = max(0, b.kv_len[i]);
    return s;
}

}  // namespace emb
