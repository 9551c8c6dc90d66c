// kv4_prompt.cuh — attention over the paged 4-bit KV cache, many rows per sequence.
//
// The same mathematics as kv4_attn.cuh with 128 query rows (tokens x the query heads
// of a kv head) against tiles of 64 positions on tcgen05, one CTA per (row tile, kv
// head, sequence), two CTAs on an SM so that one's softmax runs under the other's
// products. Warps have roles:
//   0-3  softmax: a thread owns a row; it reads the row's 64 scores from tensor memory,
//        raises the maximum if a score passes it by 2^8 (then O is rescaled in tensor
//        memory, which is rare), and writes the weights over the scores
//   4,5  keys, 6,7 values: packed codes from global memory to exact fp16 numbers
//        (code - 8) * d in shared memory, swizzled as the products read them; the
//        values are transposed on the way, so both operands are K-major
//   4    its first lane also issues the products: S = Q K^T, two tiles in turn, O += P V
//        with P from tensor memory (a ninth warp for it would leave 96 registers a thread)
// fp32 queries and weights enter as an fp16 rounding and its rest (two products into
// the same sums, 22 bits); fp16 queries are exact as they are, and their weights are
// rounded to 11 bits, which changes an output by less than its own rounding does.
#pragma once

#include "kv4_attn.cuh"

namespace emb {

constexpr int KP_THREADS = 256, KP_ROWS = 128, KP_POS = 64;
constexpr unsigned long long KP_WAIT_NS = 1000000000ull;

template <typename T, int HD>
struct KpLayout {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;    // fp16 parts of a query and of a weight
    static constexpr int PANELS = (HD + 63) / 64;           // panels of 64 fp16 (128 bytes) of a row
    static constexpr int Q_PART = PANELS * KP_ROWS * 128, K_BYTES = PANELS * KP_POS * 128, V_BYTES = HD * 128;
    static constexpr int OFF_K = PARTS * Q_PART, OFF_V = OFF_K + K_BYTES, OFF_X = OFF_V + V_BYTES;
    static constexpr int SMEM = OFF_X + 1024;               // + slack to align the base to 1024
    static constexpr int COLS = 256, COL_O = 128;           // tensor memory: S / P of two tiles, then O
};

struct KpShared {
    uint64_t k_full, k_empty, v_full, v_empty, s_full[2], p_full[2];
    uint32_t tmem;
    int abort;
    uint64_t valid[4];          // which positions of a tile there are, by tile number mod 4
    float rscale[KP_ROWS];
};

// Wait for a phase; gives up after KP_WAIT_NS or as soon as another role has given up,
// so that a product that never completes ends the CTA (its rows become NaN).
EMB_DEV bool kp_wait(uint64_t *bar, uint32_t parity, volatile int *abort) {
    if (mbar_try_wait(bar, parity)) return true;
    unsigned long long t0, t1;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    while (!mbar_try_wait(bar, parity)) {
        if (*abort) return false;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t1));
        if (t1 - t0 > KP_WAIT_NS) {
            *abort = 1;
            return false;
        }
    }
    return true;
}

EMB_DEV void kp_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
EMB_DEV void kp_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
EMB_DEV void kp_fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// K-major operand in shared memory, rows of 128 bytes with 128-byte swizzle
EMB_DEV uint64_t kp_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// byte of 16-byte chunk c of row r inside a panel
EMB_DEV uint32_t kp_chunk(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// D[tmem] (+)= A * B^T, fp16 operands, fp32 sums, K = 16; A from shared or tensor memory
EMB_DEV void kp_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
EMB_DEV void kp_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
EMB_DEV void kp_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// 32 (16) consecutive columns of this thread's lane
template <int I, int N>
EMB_DEV void kp_ld32(float (&r)[N], uint32_t ta) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[I + 0]), "=f"(r[I + 1]), "=f"(r[I + 2]), "=f"(r[I + 3]), "=f"(r[I + 4]), "=f"(r[I + 5]), "=f"(r[I + 6]), "=f"(r[I + 7]), "=f"(r[I + 8]), "=f"(r[I + 9]), "=f"(r[I + 10]), "=f"(r[I + 11]), "=f"(r[I + 12]), "=f"(r[I + 13]), "=f"(r[I + 14]), "=f"(r[I + 15]), "=f"(r[I + 16]), "=f"(r[I + 17]), "=f"(r[I + 18]), "=f"(r[I + 19]), "=f"(r[I + 20]), "=f"(r[I + 21]), "=f"(r[I + 22]), "=f"(r[I + 23]), "=f"(r[I + 24]), "=f"(r[I + 25]), "=f"(r[I + 26]), "=f"(r[I + 27]), "=f"(r[I + 28]), "=f"(r[I + 29]), "=f"(r[I + 30]), "=f"(r[I + 31])
        : "r"(ta)
        : "memory");
}
EMB_DEV void kp_st16(uint32_t ta, const uint32_t (&u)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(ta),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
        : "memory");
}
EMB_DEV void kp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// the lower (1024 + c) and upper (1024 + 16 c) nibbles' exact (code - 8) * d
EMB_DEV uint32_t kp_low(uint32_t w, __half2 d) {
    return h2bits(__hmul2(__hsub2(bits_h2(and_or(w, 0x000F000Fu, 0x64006400u)), bits_h2(0x64086408u)), d));
}
EMB_DEV uint32_t kp_high(uint32_t w, __half2 d) {
    return h2bits(__hmul2(
        __hfma2(bits_h2(and_or(w, 0x00F000F0u, 0x64006400u)), bits_h2(0x2C002C00u), bits_h2(0xD480D480u)), d));
}

// tiles of KP_POS positions that a row tile sees
struct KpRange {
    int sink_tiles, lo, total;
    __device__ __forceinline__ int pos(int j) const { return (j < sink_tiles ? j : j + (lo - sink_tiles)) * KP_POS; }
};
EMB_DEV KpRange kp_range(int first_pos, int last_pos, int len, int window, int sinks) {
    KpRange r;
    const int stop = max(0, min(len, last_pos + 1)), end = (stop + KP_POS - 1) / KP_POS;
    const long long from = window > 0 ? (long long)first_pos - window + 1 : 0;
    r.lo = (int)max(0ll, min(from, (long long)stop)) / KP_POS;
    r.sink_tiles = min((int)(((long long)sinks + KP_POS - 1) / KP_POS), r.lo);
    r.total = r.sink_tiles + end - r.lo;
    return r;
}

template <typename T, int HD>
__global__ void __launch_bounds__(KP_THREADS, 2) kv4_prompt_kernel(const Kv4AttnArgs a) {
    using L = KpLayout<T, HD>;
    constexpr int NB = HD / 32, GB = kv4_group(HD), PARTS = L::PARTS;
    extern __shared__ uint8_t kp_raw[];
    __shared__ KpShared sh;
    const uint32_t raw = smem_u32(kp_raw);
    uint8_t *sm = kp_raw + ((1024u - (raw & 1023u)) & 1023u);
    const uint32_t sm32 = smem_u32(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int seq = blockIdx.z, kv = blockIdx.y;
    const Kv4Seq s = kv4_seq(a.b, seq);
    const int rows = min(s.rows, a.max_q) * a.group;
    // the latest rows see the most positions: they go first
    const int row_first = ((int)gridDim.x - 1 - (int)blockIdx.x) * KP_ROWS;
    if (row_first >= rows) return;
    const int pos0 = s.len - s.rows, len = min(min(s.len, a.max_kv), a.b.cap);
    const int first_pos = pos0 + row_first / a.group,
              last_pos = pos0 + (min(rows, row_first + KP_ROWS) - 1) / a.group;
    const KpRange range = kp_range(first_pos, last_pos, len, a.window, a.sinks);
    const int n = range.total;

    if (tid == 0) {
        mbar_init(&sh.k_full, 64);
        mbar_init(&sh.k_empty, 1);
        mbar_init(&sh.v_full, 64);
        mbar_init(&sh.v_empty, 1);
        for (int i = 0; i < 2; i++) { mbar_init(&sh.s_full[i], 1); mbar_init(&sh.p_full[i], 128); }
        fence_mbar_init();
        sh.abort = 0;
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"((uint32_t)L::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    {
        // queries: a warp takes 16 rows; within 8 dims the order is 0,4,1,5,2,6,3,7, as
        // the keys come out of their words
        for (int i = 0; i < KP_ROWS / 8; i++) {
            const int r = warp * (KP_ROWS / 8) + i, rr = row_first + r;
            float v[NB], m = 0.0f;
            bool finite = true;
            const int tok = rr / a.group, h = kv * a.group + rr - tok * a.group;
            const T *src = (const T *)a.q + (int64_t)(s.row0 + tok) * a.q_tok + h * a.q_head + lane;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                v[b] = rr < rows ? widen(src[b * 32]) : 0.0f;
                finite = finite && fabsf(v[b]) < INFINITY;
                m = fmaxf(m, fabsf(v[b]));
            }
            m = warp_max(m);
            finite = __all_sync(0xffffffffu, finite);
            // |q| * 2^e below 2^14; the sign of the scale goes into the queries, so that
            // a row's largest product is its largest score
            const int e = m > 0.0f ? 13 - ilogbf(m) : 0;
            float f1 = __int_as_float((127 + e / 2) << 23);
            const float f2 = __int_as_float((127 + e - e / 2) << 23);
            // (never 0: a hidden score, -inf, must stay -inf)
            if (lane == 0)
                sh.rscale[r] = a.scale == 0.0f ? 1.0f : fmaxf(fabsf(a.scale) * KV4_LOG2E / f1 / f2, 1.2e-38f);
            if (a.scale < 0.0f) f1 = -f1;
            if (a.scale == 0.0f) f1 = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float y = finite ? v[b] * f1 * f2 : __int_as_float(0x7fffffff);
                const int d = b * 32 + lane, c = d >> 3, k = d & 7, p = k < 4 ? 2 * k : 2 * k - 7;
                const uint32_t at = (c >> 3) * (KP_ROWS * 128) + kp_chunk(r, c & 7) + 2 * p;
                const __half hi = __float2half_rn(y);
                *reinterpret_cast<__half *>(sm + at) = hi;
                if (PARTS == 2)
                    *reinterpret_cast<__half *>(sm + L::Q_PART + at) = __float2half_rn(y - __half2float(hi));
            }
        }
        kp_fence_smem();
    }
    kp_fence_before();
    __syncthreads();
    kp_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int *abort = &sh.abort;

    if (warp < 4) {
        // ---------------------------------------------------------- softmax ----
        const int r = tid, rr = row_first + r, pos = pos0 + min(rr, rows - 1) / a.group;
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
        const float rs = sh.rscale[r];
        // positions that every row sees: up to the first row's, from the last row's window on
        const long long all_from = a.window > 0 ? (long long)last_pos - a.window + 1 : 0;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < n; j++) {
            ok = kp_wait(&sh.s_full[j & 1], (j >> 1) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            kp_fence_after();
            const uint32_t at = mine + (j & 1) * 64;
            float v[64];
            kp_ld32<0>(v, at);
            kp_ld32<32>(v, at + 32);
            const int p0 = range.pos(j);
            const uint64_t valid = sh.valid[j & 3];
            if (!(p0 >= all_from && p0 + KP_POS - 1 <= first_pos && valid == ~0ull)) {
                // bit p: the row sees position p0 + p
                uint64_t see = 0;
                const int upto = pos - p0;                           // p <= upto
                if (upto >= 0) see = upto >= 63 ? ~0ull : (2ull << upto) - 1;
                if (a.window > 0) {
                    const long long from = (long long)pos - a.window + 1 - p0;   // p >= from, or a sink
                    uint64_t keep = from <= 0 ? ~0ull : from >= 64 ? 0ull : ~0ull << from;
                    const long long sk = (long long)a.sinks - p0;
                    keep |= sk <= 0 ? 0ull : sk >= 64 ? ~0ull : (1ull << sk) - 1;
                    see &= keep;
                }
                see &= valid;
                const uint32_t s0 = (uint32_t)see, s1 = (uint32_t)(see >> 32);
#pragma unroll
                for (int p = 0; p < 32; p++) {
                    if (!((s0 >> p) & 1)) v[p] = -INFINITY;
                    if (!((s1 >> p) & 1)) v[32 + p] = -INFINITY;
                }
            }
            float mx = v[0];
#pragma unroll
            for (int p = 1; p < 64; p++) mx = fmaxf(mx, v[p]);
            mx *= rs;
            if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
                const float mn = fmaxf(m, mx);
                const float f = mn == m ? 1.0f : kv4_exp2(m - mn);
                m = mn;
                l *= f;
                if (j > 0) {
                    ok = kp_wait(&sh.v_empty, (j - 1) & 1, abort);   // the products into O so far
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    kp_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        kp_ld32<0>(o, mine + L::COL_O + c);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t u[16];
#pragma unroll
                            for (int k = 0; k < 16; k++) u[k] = __float_as_uint(o[16 * h + k] * f);
                            kp_st16(mine + L::COL_O + c + 16 * h, u);
                        }
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : m - 6.0f;
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float e0 = kv4_exp2(fmaf(v[h * 32 + 2 * k], rs, -base));
                    const float e1 = kv4_exp2(fmaf(v[h * 32 + 2 * k + 1], rs, -base));
                    sum += e0 + e1;
                    hi[k] = pack_half2(e0, e1);
                    if (PARTS == 2) {
                        const float2 q = __half22float2(bits_h2(hi[k]));
                        lo[k] = pack_half2(e0 - q.x, e1 - q.y);
                    }
                }
                kp_st16(at + h * 16, hi);
                if (PARTS == 2) kp_st16(at + 32 + h * 16, lo);
            }
            l += sum;
            kp_wait_st();
            kp_fence_before();
            mbar_arrive(&sh.p_full[j & 1]);
        }
        if (n > 0 && ok) {
            ok = kp_wait(&sh.v_empty, (n - 1) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            kp_fence_after();
        }
        const bool live = rr < rows;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int tok = min(rr, rows - 1) / a.group, h = kv * a.group + min(rr, rows - 1) - tok * a.group;
        T *out = (T *)a.out + (int64_t)(s.row0 + tok) * a.out_tok + h * a.out_head;
        const bool vec = !((uintptr_t)a.out % 16 || (a.out_tok * sizeof(T)) % 16 || (a.out_head * sizeof(T)) % 16);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
            float o[32];
            if (n > 0 && ok) kp_ld32<0>(o, mine + L::COL_O + c);
#pragma unroll
            for (int k = 0; k < 32; k++) o[k] = !ok ? __int_as_float(0x7fffffff) : l == 0.0f ? 0.0f : o[k] * inv;
            if (!live) continue;
            if (vec && sizeof(T) == 4) {
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                    *reinterpret_cast<float4 *>(out + c + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            } else if (vec) {
#pragma unroll
                for (int k = 0; k < 32; k += 8)
                    *reinterpret_cast<uint4 *>(out + c + k) =
                        make_uint4(pack_half2(o[k], o[k + 1]), pack_half2(o[k + 2], o[k + 3]),
                                   pack_half2(o[k + 4], o[k + 5]), pack_half2(o[k + 6], o[k + 7]));
            } else {
#pragma unroll
                for (int k = 0; k < 32; k++) kv_round(o[k], &out[c + k]);
            }
        }
        kp_fence_before();
    } else {
        // --------------------------------------- keys and values, products ----
        const bool keys = warp < 6;
        const int t64 = (tid - 128) & 63, ps = 1 << a.c.page_shift;
        const int32_t *table = a.b.table + (size_t)seq * a.b.table_stride;
        const uint8_t *base = a.c.data + (size_t)kv * a.c.chunk;
        const uint64_t stride = (uint64_t)a.c.n_kv * a.c.chunk;
        uint8_t *dst = sm + (keys ? L::OFF_K : L::OFF_V);
        // page of position p (-1: none), asked for two tiles ahead; its group of 16, or null
        auto page_at = [&](int j, int in_tile) {
            const int p = range.pos(j) + in_tile;
            return j < n && p < len ? __ldg(table + (p >> a.c.page_shift)) : -1;
        };
        auto group = [&](int page, int p) -> const uint8_t * {
            if ((unsigned)page >= (unsigned)a.c.n_pages) return nullptr;
            return base + (uint64_t)(uint32_t)page * stride + ((p & (ps - 1)) >> 4) * GB;
        };
        const bool issuer = tid == 128;
        constexpr uint32_t kind = 1u << 4 | (uint32_t)(KP_ROWS >> 4) << 24;      // fp16 x fp16 -> fp32, M = 128
        constexpr uint32_t idesc_s = kind | (uint32_t)(KP_POS >> 3) << 17, idesc_o = kind | (uint32_t)(HD >> 3) << 17;
        auto scores = [&](int j) {
            kp_fence_after();
            const uint32_t d = tmem + (j & 1) * 64;
#pragma unroll
            for (int q = 0; q < PARTS; q++)
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
                    kp_mma_ss(d, kp_desc(sm32 + q * L::Q_PART + (k >> 2) * (KP_ROWS * 128) + (k & 3) * 32),
                              kp_desc(sm32 + L::OFF_K + (k >> 2) * (KP_POS * 128) + (k & 3) * 32), idesc_s, q + k > 0);
            kp_commit(&sh.s_full[j & 1]);
            kp_commit(&sh.k_empty);
        };
        auto outputs = [&](int j) {
            kp_fence_after();
            const uint32_t p = tmem + (j & 1) * 64;
#pragma unroll
            for (int q = 0; q < PARTS; q++)
#pragma unroll
                for (int k = 0; k < KP_POS / 16; k++)
                    kp_mma_ts(tmem + L::COL_O, p + q * 32 + k * 8, kp_desc(sm32 + L::OFF_V + k * 32), idesc_o,
                              j > 0 || q + k > 0);
            kp_commit(&sh.v_empty);
        };
        int done = 0;                     // tiles whose products into O were issued
        bool fine = true;
        // A tile's packed words are loaded while the tile before is made operands.
        // keys: word column t of the positions half*32 + 8 i + low; values: words g of the
        // positions 8 c ..
        const int t = (t64 >> 3) & 3, half = t64 >> 5, low = t64 & 7, c = t64 & 7, g = t64 >> 3;
        uint32_t nw[4][NB], nd[4][NB];
        int pg[2] = {-1, -1};
        auto pages = [&](int j) {
            if (keys) {
                pg[0] = page_at(j, half * 32);
                pg[1] = page_at(j, half * 32 + 16);
            } else {
                pg[0] = page_at(j, (c >> 1) * 16);
            }
        };
        uint32_t nok = 0;                 // keys: which of the four positions there are
        auto load = [&](int j) {
            const int p0 = range.pos(j);
            nok = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int b = 0; b < NB; b++) nw[i][b] = nd[i][b] = 0;
            }
            if (j >= n) return;
            if (keys) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int p = half * 32 + i * 8 + low, r = p & 15;
                    const uint8_t *gr = group(pg[i >> 1], p0 + p);
                    if (!gr) continue;
                    lds_words<NB>(nw[i], gr + r * (HD / 2) + t * (4 * NB));
                    uint32_t ks[NB < 2 ? 1 : NB / 2];
                    lds_words<NB / 2>(ks, gr + 16 * HD + r * (2 * NB));
#pragma unroll
                    for (int b = 0; b < (NB < 2 ? 1 : NB / 2); b++) nd[i][b] = ks[b];
                    if (p0 + p < len) nok |= 1u << (i * 8 + low);
                }
            } else {
                const uint8_t *gr = group(pg[0], p0 + (c >> 1) * 16);
                if (!gr) return;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int pair = (c & 1) * 4 + i;
                    lds_words<NB>(nw[i], gr + 8 * HD + pair * HD + g * (4 * NB));
                    lds_words<NB>(nd[i], gr + 16 * HD + 32 * NB + pair * (4 * NB));
                }
            }
        };
        pages(0);
        load(0);
        pages(1);
        for (int j = 0; j < n; j++) {
            uint32_t w[4][NB], d[4][NB];
            const uint32_t ok = nok;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int b = 0; b < NB; b++) { w[i][b] = nw[i][b]; d[i][b] = nd[i][b]; }
            load(j + 1);
            pages(j + 2);
            const int p0 = range.pos(j);
            if (keys) {
                // the tile's positions, as a mask (both warps have a half)
                const uint32_t bits = __reduce_or_sync(0xffffffffu, ok);
                if (!__all_sync(0xffffffffu, j == 0 || kp_wait(&sh.k_empty, (j - 1) & 1, abort))) break;
                if (lane == 0) reinterpret_cast<uint32_t *>(&sh.valid[j & 3])[half] = bits;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int p = half * 32 + i * 8 + low;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const __half2 dd = bits_h2(__byte_perm(d[i][b / 2], 0, (b & 1) ? 0x3232 : 0x1010));
                        const uint32_t x = w[i][b], y = x >> 8;
                        const uint4 q = make_uint4(kp_low(x, dd), kp_high(x, dd), kp_low(y, dd), kp_high(y, dd));
                        *reinterpret_cast<uint4 *>(dst + (b >> 1) * (KP_POS * 128) + kp_chunk(p, 4 * (b & 1) + t)) = q;
                    }
                }
                kp_fence_smem();
                mbar_arrive(&sh.k_full);
                if (issuer && fine) {
                    fine = kp_wait(&sh.k_full, j & 1, abort);
                    // the weights that tile j - 2 left where these scores go have been used
                    if (fine && j > 1) fine = kp_wait(&sh.v_empty, j & 1, abort);
                    if (fine) scores(j);
                    if (fine && j > 0) {
                        fine = kp_wait(&sh.p_full[(j - 1) & 1], ((j - 1) >> 1) & 1, abort) &&
                               kp_wait(&sh.v_full, (j - 1) & 1, abort);
                        if (fine) {
                            outputs(j - 1);
                            done = j;
                        }
                    }
                }
                __syncwarp();
            } else {
                // positions behind the length may hold any bytes: their scales count as 0
                if (p0 + KP_POS > len) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int left = len - (p0 + 8 * c + 2 * i);
                        const uint32_t keep = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0x0000FFFFu : 0u;
#pragma unroll
                        for (int b = 0; b < NB; b++) d[i][b] &= keep;
                    }
                }
                if (!__all_sync(0xffffffffu, j == 0 || kp_wait(&sh.v_empty, (j - 1) & 1, abort))) break;
#pragma unroll
                for (int b = 0; b < NB; b++) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t x[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t u = k < 2 ? w[i][b] : w[i][b] >> 8;
                            x[i] = (k & 1) ? kp_high(u, bits_h2(d[i][b])) : kp_low(u, bits_h2(d[i][b]));
                        }
                        *reinterpret_cast<uint4 *>(dst + kp_chunk(b * 32 + 4 * g + k, c)) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                kp_fence_smem();
                mbar_arrive(&sh.v_full);
            }
        }
        if (issuer && n > 0) {
            fine = fine && kp_wait(&sh.p_full[(n - 1) & 1], ((n - 1) >> 1) & 1, abort) &&
                   kp_wait(&sh.v_full, (n - 1) & 1, abort);
            if (fine) {
                outputs(n - 1);
                done = n;
            }
            // products in flight end before tensor memory is given back
            int never = 0;
            if (done > 0) kp_wait(&sh.v_empty, (done - 1) & 1, &never);
            if (done < n) {               // given up: a last commit covers the scores too
                kp_commit(&sh.v_empty);
                kp_wait(&sh.v_empty, done & 1, &never);
            }
        }
    }
    __syncwarp();
    __syncthreads();
    kp_fence_after();
    if (warp == 4)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::COLS) : "memory");
}

// ------------------------------------------------------------------- host ----

template <typename T, int HD>
static int kv4_prompt_launch(const Kv4AttnArgs &a, cudaStream_t st) {
    using L = KpLayout<T, HD>;
    static std::atomic<unsigned long long> ready{0};      // devices whose limit is raised
    int dev = 0;
    CK(cudaGetDevice(&dev));
    if (dev >= 64 || !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        CK(cudaFuncSetAttribute(kv4_prompt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const long long tiles = ((long long)a.max_q * a.group + KP_ROWS - 1) / KP_ROWS;
    if (tiles > 0x7FFFFFFF) return set_err("kv4 attention: max_q %d is too large", a.max_q);
    const dim3 grid((unsigned)tiles, (unsigned)a.c.n_kv, (unsigned)a.b.n_seqs);
    kv4_prompt_kernel<T, HD><<<grid, KP_THREADS, L::SMEM, st>>>(a);
    CK(cudaGetLastError());
    return 0;
}

template <typename T>
static int kv4_prompt_hd(const Kv4AttnArgs &a, int hd, cudaStream_t st) {
    switch (hd) {
    case 32: return kv4_prompt_launch<T, 32>(a, st);
    case 64: return kv4_prompt_launch<T, 64>(a, st);
    default: return kv4_prompt_launch<T, 128>(a, st);
    }
}

}  // namespace emb
