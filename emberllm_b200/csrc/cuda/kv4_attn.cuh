// kv4_attn.cuh — attention over the paged 4-bit KV cache.
//
// Per row at position pos and per query head: s_p = scale * (q . k_p) over the
// visible positions p, weights exp(s_p - m) with m the largest visible s_p, and
// out = sum weights_p * v_p / sum weights_p, in one pass over the cache: when a
// larger score appears, what was summed so far is multiplied by exp(m_old - m_new).
#pragma once

#include "kv4.cuh"
#include "runtime_internal.cuh"

namespace emb {

struct Kv4AttnArgs {
    Kv4View c;
    Kv4Rows b;
    const void *q;
    void *out;
    int64_t q_tok, q_head, out_tok, out_head;
    int n_heads, group;
    float scale;
    int max_kv, max_q, window, sinks;
    float *ws;
};

EMB_DEV bool kv4_visible(int pos, int p, int window, int sinks) {
    return p <= pos && (window == 0 || pos - p < window || p < sinks);
}

static inline size_t kv4_attention_workspace(int, int, int, int, int, int) { return 0; }

// One warp per (row, query head): each lane holds hd/32 dims of the query and of
// the output, the score is summed over the warp.
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv4_attn_row_kernel(Kv4AttnArgs a) {
    constexpr int NB = HD / 32;
    const Kv4Seq s = kv4_seq(a.b, blockIdx.z);
    const int head = blockIdx.y, lane = threadIdx.x & 31;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= s.rows) return;
    const int len = min(s.len, a.max_kv);
    const int pos = s.len - s.rows + row;
    const T *q = (const T *)a.q + (int64_t)(s.row0 + row) * a.q_tok + head * a.q_head;
    float qv[NB], o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        qv[b] = widen(q[b * 32 + lane]) * a.scale;
        o[b] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int ps = 1 << a.c.page_shift;
    for (int p = 0; p < len && p <= pos; p++) {
        if (!kv4_visible(pos, p, a.window, a.sinks)) continue;
        const int page = kv4_page(a.c, a.b, blockIdx.z, p);
        if (page < 0) continue;
        const uint8_t *ch = kv4_chunk_ptr(a.c, page, head / a.group);
        const int slot = p & (ps - 1);
        const __half *ks = reinterpret_cast<const __half *>(ch + (size_t)ps * HD) + slot * NB;
        const __half *vs = ks + ps * NB;
        const uint8_t *kr = ch + (size_t)slot * (HD / 2), *vr = kr + (size_t)ps * (HD / 2);
        float sc = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int byte = kr[(lane >> 3) * (4 * NB) + 4 * b + ((lane & 7) >> 1)];
            const int code = (lane & 1) ? byte >> 4 : byte & 15;
            sc = fmaf(qv[b], (float)(code - 8) * __half2float(ks[b]), sc);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sc += __shfl_xor_sync(0xffffffffu, sc, off);
        const float mn = fmaxf(m, sc);
        const float f = m == mn ? 1.0f : __expf(m - mn), w = __expf(sc - mn);
        m = mn;
        l = fmaf(l, f, w);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int byte = vr[(lane >> 2) * (2 * NB) + 2 * b + ((lane >> 1) & 1)];
            const int code = (lane & 1) ? byte >> 4 : byte & 15;
            o[b] = fmaf(o[b], f, w * ((float)(code - 8) * __half2float(vs[b])));
        }
    }
    T *out = (T *)a.out + (int64_t)(s.row0 + row) * a.out_tok + head * a.out_head;
#pragma unroll
    for (int b = 0; b < NB; b++) kv_round(l == 0.0f ? 0.0f : o[b] / l, &out[b * 32 + lane]);
}

template <typename T>
static int kv4_attention_launch(const Kv4AttnArgs &a, int hd, cudaStream_t st) {
    const dim3 grid((unsigned)((a.max_q + 3) / 4), (unsigned)a.n_heads, (unsigned)a.b.n_seqs);
    switch (hd) {
    case 32: kv4_attn_row_kernel<T, 32><<<grid, 128, 0, st>>>(a); break;
    case 64: kv4_attn_row_kernel<T, 64><<<grid, 128, 0, st>>>(a); break;
    default: kv4_attn_row_kernel<T, 128><<<grid, 128, 0, st>>>(a); break;
    }
    CK(cudaGetLastError());
    return 0;
}

}  // namespace emb
