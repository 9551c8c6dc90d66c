// kv4_attn.cuh — attention over the paged 4-bit KV cache, few rows per sequence.
//
// Per row at position pos and per query head: s_p = scale * (q . k_p) over the
// visible positions p, weights exp(s_p - m) with m the largest visible s_p, and
// out = sum weights_p * v_p / sum weights_p, in one pass over the cache: when a
// larger score appears, what was summed so far is multiplied by exp(m_old - m_new).
//
// Bound by memory (144 bytes a position and kv head of 128) once the codes are
// turned into matrix operands cheaply enough: at 44 bytes per ns and SM there are
// about 3 lane instructions per element. So the codes stay packed until they are in
// registers, in the order of the fragments of mma m16n8k16, and become operands
// there; in shared memory, as tcgen05 wants them, they would be 4x the bytes, and
// with a handful of query rows per kv head its 64 rows and more have nothing to do
// (prompts use it). Asynchronous copies keep a unit ahead in flight per warp without
// holding registers for it.
//   scores   A = keys (16 positions x 16 dims), the whole numbers code - 8 as fp16: a
//        nibble or-ed into the mantissa of 1024 (or, in place, its sixteenfold), less 1032
//        (1/16 of it less 72); B = queries. Sums per 32-block, to which the block's scale
//        is applied in fp32. (A masked nibble is an fp16 subnormal already, code * 2^-24,
//        and -8 * (sum of the queries) can be added afterwards: 8 instructions in 28 fewer,
//        but the larger sums cost the result two bits, 3e-6 instead of 4e-7 of it.)
//   outputs  A = values (16 dims x 16 positions), made exact fp16 numbers
//        (code - 8) * d; B = the weights.
// Queries and weights take two columns of B each, the fp16 rounding and the
// rounded rest: 22 bits for the price of idle columns. A query row is first scaled
// by a power of two so that its largest element is below 2^14.
//
// 64 sequences of 200-1600 positions, 16 / 8 heads of 128, fp32: 28.7 us, 2.4 TB/s, issue slots half
// used (the longest sequences end alone); two of 37-41k: 30.8 us, 26.0 without the join, issue 61 %.
#pragma once

#include <atomic>

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
    int chunks;                   // row chunks per kv head
    int span, parts;              // units of a CTA; CTAs of the longest sequence
    float *ws;
};

constexpr int KD_WARPS = 4;
constexpr int KD_THREADS = 32 * KD_WARPS;
constexpr int KD_UNIT = 32;        // positions a warp takes at a time, in two groups of 16
constexpr float KV4_LOG2E = 1.44269504088896341f;

EMB_DEV bool kv4_visible(int pos, int p, int window, int sinks) {
    return p <= pos && (window == 0 || pos - p < window || p < sinks);
}

// [sinks, this] are the positions in front of every row's window when the first row is
// at `first`; hidden from all rows, they may never have been written
EMB_DEV int kv4_before(int first, int window) {
    return window > 0 ? (int)max(-1ll, (long long)first - window) : -1;
}

EMB_DEV float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// D = A (16x16) * B (16x8) + C, fp16 operands, fp32 sums
EMB_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                     float c0, float c1, float c2, float c3) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

EMB_DEV uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
EMB_DEV __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
EMB_DEV uint32_t pack_half2(float lo, float hi) { return h2bits(__floats2half2_rn(lo, hi)); }
// (v & mask) | magic as the one instruction it can be: written in C++ it became two,
// a tenth of the kernel's instructions
EMB_DEV uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(magic));
    return r;
}

// code - 8 of a word's lower (upper) nibbles of each byte 0 and 2, exact
EMB_DEV uint32_t kd_low(uint32_t w) {
    return h2bits(__hsub2(bits_h2(and_or(w, 0x000F000Fu, 0x64006400u)), bits_h2(0x64086408u)));
}
EMB_DEV uint32_t kd_high(uint32_t w) {
    return h2bits(__hfma2(bits_h2(and_or(w, 0x00F000F0u, 0x64006400u)), bits_h2(0x2C002C00u), bits_h2(0xD480D480u)));
}

// W consecutive 32-bit words of shared memory (W = 0: one 16-bit piece)
template <int W>
EMB_DEV void lds_words(uint32_t (&r)[W < 1 ? 1 : W], const uint8_t *p) {
    if (W == 0) r[0] = *reinterpret_cast<const uint16_t *>(p);
    else if (W == 1) r[0] = *reinterpret_cast<const uint32_t *>(p);
    else if (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r[0] = v.x; r[W - 1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        r[0] = v.x; r[1 % W] = v.y; r[2 % W] = v.z; r[W - 1] = v.w;
    }
}

// the units of KD_UNIT positions a sequence's rows see: those of the sinks, then
// those from the first row's window on
struct KdRange {
    int sink_units, lo, total;
    // first position of unit i
    __device__ __forceinline__ int pos(int i) const { return (i < sink_units ? i : i + (lo - sink_units)) * KD_UNIT; }
};
EMB_DEV KdRange kd_range(int first_pos, int last_pos, int len, int window, int sinks) {
    KdRange r;
    const int stop = max(0, min(len, last_pos + 1)), end = (stop + KD_UNIT - 1) / KD_UNIT;
    const long long from = window > 0 ? (long long)first_pos - window + 1 : 0;
    r.lo = (int)max(0ll, min(from, (long long)stop)) / KD_UNIT;
    r.sink_units = min((int)(((long long)sinks + KD_UNIT - 1) / KD_UNIT), r.lo);
    r.total = r.sink_units + end - r.lo;
    return r;
}

// An item is one (sequence, kv head, chunk of 4 * NT rows); its work is the units its
// sequence's rows see, cut into pieces of `span` units where there are too few items
// to fill the GPU. A piece is a CTA's work; kv4_join_kernel joins an item's pieces.
// (Dealing out all units in even shares, across items, was slower: 64 ragged streams
// 33 -> 35 us, 512 short and long ones 50 -> 76 us. More items then get cut, and a
// cut costs the start and end of a CTA, some 8,000 cycles; the scheduler's own
// filling of free slots does the rest as well.)
template <int HD, int NT>
struct KdLayout {
    static constexpr int STAGES = 2, R = 4 * NT;
    static constexpr int UNIT = 2 * kv4_group(HD);                      // bytes of a unit
    static constexpr int RING = KD_WARPS * STAGES * UNIT;
    static constexpr int PS = HD + 4;                                   // row stride of partials, in floats
    static constexpr int PART = KD_WARPS * R * PS * 4;                  // takes the ring's place at the end
    static constexpr int SMEM = RING > PART ? RING : PART;
    static constexpr int CTAS = NT == 1 ? (HD == 128 ? 4 : 5) : (HD == 128 ? 2 : 4);   // per SM, by registers
};
constexpr int KD_SPAN_MIN = 16;       // units of a piece, at least
constexpr int KD_MAX_SLOTS = 148 * 5; // CTAs that fit the GPU, at most

struct KdItem {
    Kv4Seq s;
    int len, pos0, rows;              // visible length, first row's position, rows (all heads of a group)
    KdRange range;
};
EMB_DEV KdItem kd_item(const Kv4AttnArgs &a, int seq) {
    KdItem it;
    it.s = kv4_seq(a.b, seq);
    it.rows = min(it.s.rows, a.max_q) * a.group;
    it.pos0 = it.s.len - it.s.rows;
    it.len = min(min(it.s.len, a.max_kv), a.b.cap);
    it.range = kd_range(it.pos0, it.pos0 + min(it.s.rows, a.max_q) - 1, it.len, a.window, a.sinks);
    return it;
}

// a piece's result: per row its max (log2 units), sum and HD outputs
template <int HD, int NT>
EMB_DEV float *kd_partial(const Kv4AttnArgs &a, int item, int piece) {
    return a.ws + ((size_t)item * a.parts + piece) * (KdLayout<HD, NT>::R * KdLayout<HD, NT>::PS);
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(KD_THREADS, KdLayout<HD, NT>::CTAS) kv4_decode_kernel(const Kv4AttnArgs a) {
    using L = KdLayout<HD, NT>;
    constexpr int NB = HD / 32, R = L::R, PS = L::PS, GB = kv4_group(HD);
    extern __shared__ __align__(128) uint8_t ring[];                    // [warp][stage][unit]
    float(*part)[R][PS] = reinterpret_cast<float(*)[R][PS]>(ring);      // [warp][row][PS]
    __shared__ __align__(16) uint4 qf[NT][NB][32];
    __shared__ __align__(16) float x[R][HD];  // scaled queries
    __shared__ float rscale[R];               // the scores' factor
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, kv = blockIdx.y / a.chunks, chunk_row = (blockIdx.y - kv * a.chunks) * R;
    const KdItem it = kd_item(a, seq);
    const int rows = it.rows - chunk_row;                   // rows of this chunk (token-major, head in group)
    const int len = it.len, pos0 = it.pos0;
    const KdRange range = it.range;
    const Kv4Seq &s = it.s;
    const int u0 = blockIdx.x * a.span, u1 = min(range.total, u0 + a.span);
    if (rows <= 0 || (u0 >= range.total && u0 > 0)) return;
    // a sequence that fits one piece is finished here
    float *partial = range.total <= a.span
                         ? nullptr
                         : kd_partial<HD, NT>(a, blockIdx.z * gridDim.y + blockIdx.y, blockIdx.x);

    // the warp's query rows, asked for before anything waits
    float qv[NT][NB];
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int rr = chunk_row + warp * NT + i, tok = rr / a.group, h = kv * a.group + rr - tok * a.group;
        const T *src = (const T *)a.q + (int64_t)(s.row0 + tok) * a.q_tok + h * a.q_head + lane;
#pragma unroll
        for (int b = 0; b < NB; b++) qv[i][b] = warp * NT + i < rows ? widen(src[b * 32]) : 0.0f;
    }

    // The warp's units are u0 + warp, + KD_WARPS, ...: the next one is copied while
    // this one is worked on, and the page numbers of the one after are loaded a unit
    // ahead and looked at when needed. A group whose page is no page is not copied;
    // its positions are hidden like those behind the length.
    const int ps = 1 << a.c.page_shift;
    const int32_t *table = a.b.table + (size_t)seq * a.b.table_stride;
    const uint8_t *base = a.c.data + (size_t)kv * a.c.chunk;
    const uint32_t stride = (uint32_t)a.c.n_kv * a.c.chunk;
    const bool small = ps == 16;                   // the groups lie in two pages
    const int last = max(0, len - 1) >> a.c.page_shift;
    struct Pages { int p[2]; };
    auto pages_of = [&](int i, int pos) {
        Pages r = {{-1, -1}};
        if (i < u1) {
            const int p = pos >> a.c.page_shift;
            r.p[0] = __ldg(table + p);
            r.p[1] = small ? __ldg(table + min(p + 1, last)) : r.p[0];
        }
        return r;
    };
    auto valid = [&](int page) { return (unsigned)page < (unsigned)a.c.n_pages; };
    uint8_t *const mine = ring + warp * (L::STAGES * L::UNIT);
    const uint32_t mine32 = smem_u32(mine) + lane * 16;
    auto copy = [&](const Pages &pg, int pos, int stage) {
        const bool ok0 = valid(pg.p[0]), ok1 = valid(pg.p[1]);
        const uint8_t *c0 = base + (uint64_t)(uint32_t)pg.p[0] * stride + (pos & (ps - 1)) / 16 * GB + lane * 16;
        const uint8_t *c1 = small ? base + (uint64_t)(uint32_t)pg.p[1] * stride + lane * 16 - GB : c0;
        const uint32_t dst = mine32 + stage * L::UNIT;
#pragma unroll
        for (int k = 0; k * 512 < L::UNIT; k++) {
            const int at = k * 512 + lane * 16;            // byte of the unit
            const bool second = at >= GB;
            if (at < L::UNIT && (second ? ok1 : ok0))
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + k * 512),
                             "l"((second ? c1 : c0) + k * 512)
                             : "memory");
        }
    };

    int i = u0 + warp, p0 = range.pos(i), pn = range.pos(i + KD_WARPS), stage = 0;
    Pages pg = pages_of(i, p0);
    if (i < u1) copy(pg, p0, 0);
    cp_async_commit();
    bool ok0 = valid(pg.p[0]), ok1 = valid(pg.p[1]);
    pg = pages_of(i + KD_WARPS, pn);
    // ---- queries into B fragments ----
    {
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int r = warp * NT + i;
            float m = 0.0f;
            bool finite = true;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                finite = finite && fabsf(qv[i][b]) < INFINITY;
                m = fmaxf(m, fabsf(qv[i][b]));
            }
            m = warp_max(m);
            finite = __all_sync(0xffffffffu, finite);
            // 2^e with m * 2^e in [2^13, 2^14), in two factors that are normal numbers
            const int e = m > 0.0f ? 13 - ilogbf(m) : 0;
            const float f1 = __int_as_float((127 + e / 2) << 23), f2 = __int_as_float((127 + e - e / 2) << 23);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float y = finite ? qv[i][b] * f1 * f2 : __int_as_float(0x7fffffff);
                x[r][b * 32 + lane] = y;
            }
            if (lane == 0)
                rscale[r] = a.scale * KV4_LOG2E * __int_as_float((127 - e / 2) << 23) *
                            __int_as_float((127 - e + e / 2) << 23);
        }
        __syncthreads();
        for (int f = warp; f < NT * NB; f += KD_WARPS) {
            // column g: row nt*4 + g/2, its fp16 rounding (even g) or the rest (odd g)
            const float *xr = x[f / NB * 4 + (g >> 1)] + (f % NB) * 32 + 8 * t;
            const float4 xa = *reinterpret_cast<const float4 *>(xr), xb = *reinterpret_cast<const float4 *>(xr + 4);
            float y[8] = {xa.x, xa.y, xa.z, xa.w, xb.x, xb.y, xb.z, xb.w};
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const float hi = __half2float(__float2half_rn(y[n]));
                y[n] = (g & 1) ? y[n] - hi : hi;
            }
            qf[f / NB][f % NB][lane] = make_uint4(pack_half2(y[0], y[4]), pack_half2(y[1], y[5]),
                                                  pack_half2(y[2], y[6]), pack_half2(y[3], y[7]));
        }
        __syncthreads();
    }

    float m[NT], l[NT], o[NT][HD / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = -INFINITY;
        l[nt] = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[nt][i][j] = 0.0f;
    }
    const float rest = (g & 1) ? -1.0f : 0.0f;             // odd columns hold what fp16 rounded away
    int row_pos[NT];
    float row_scale[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        row_pos[nt] = pos0 + (chunk_row + nt * 4 + t) / a.group;
        row_scale[nt] = rscale[nt * 4 + t];
    }
    // positions that every row sees: up to the first row's, from the last row's window on
    const int all_to = min(len, pos0 + chunk_row / a.group + 1);
    const long long all_from = a.window > 0 ? (long long)pos0 + (chunk_row + min(rows, R) - 1) / a.group - a.window + 1 : 0;
    const int before = kv4_before(pos0 + chunk_row / a.group, a.window);

    for (; i < u1; i += KD_WARPS) {
        if (i + KD_WARPS < u1) copy(pg, pn, stage ^ 1);
        cp_async_commit();
        const bool n0 = valid(pg.p[0]), n1 = valid(pg.p[1]);
        const int p2 = range.pos(i + 2 * KD_WARPS);
        pg = pages_of(i + 2 * KD_WARPS, p2);
        cp_async_wait_1();
        __syncwarp();
        const uint8_t *unit = mine + stage * L::UNIT;

        // scores of positions p0 + 16 h + g (and + 8) for row nt*4 + t
        float sc[NT][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t *kp = unit + h * GB + g * (HD / 2) + t * (4 * NB), *sp = unit + h * GB + 16 * HD + g * (2 * NB);
            uint32_t k[2][NB], ks[2][NB < 2 ? 1 : NB / 2];
            lds_words<NB>(k[0], kp);
            lds_words<NB>(k[1], kp + 8 * (HD / 2));
            lds_words<NB / 2>(ks[0], sp);
            lds_words<NB / 2>(ks[1], sp + 8 * (2 * NB));
#pragma unroll
            for (int nt = 0; nt < NT; nt++) sc[nt][2 * h] = sc[nt][2 * h + 1] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t w0 = k[0][b], w1 = k[1][b];
                const uint32_t h0 = w0 >> 8, h1 = w1 >> 8;
                const uint32_t a0 = kd_low(w0), a1 = kd_low(w1), a2 = kd_high(w0), a3 = kd_high(w1);
                const uint32_t e0 = kd_low(h0), e1 = kd_low(h1), e2 = kd_high(h0), e3 = kd_high(h1);
                const float d0 = (b & 1) ? __high2float(bits_h2(ks[0][b / 2])) : __low2float(bits_h2(ks[0][b / 2]));
                const float d1 = (b & 1) ? __high2float(bits_h2(ks[1][b / 2])) : __low2float(bits_h2(ks[1][b / 2]));
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const uint4 f = qf[nt][b][lane];
                    float c[4];
                    mma_f16(c, a0, a1, a2, a3, f.x, f.y, 0.0f, 0.0f, 0.0f, 0.0f);
                    mma_f16(c, e0, e1, e2, e3, f.z, f.w, c[0], c[1], c[2], c[3]);
                    sc[nt][2 * h] = fmaf(d0, c[0] + c[1], sc[nt][2 * h]);
                    sc[nt][2 * h + 1] = fmaf(d1, c[2] + c[3], sc[nt][2 * h + 1]);
                }
            }
        }
        const bool whole = p0 >= all_from && p0 + KD_UNIT <= all_to && ok0 && ok1;

        // softmax: the row's lanes are those of equal t
        uint32_t pb[NT][2][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int j = 0; j < 4; j++) sc[nt][j] *= row_scale[nt];
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int p = p0 + g + 8 * j;
                    if (!((j < 2 ? ok0 : ok1) && p < len && kv4_visible(row_pos[nt], p, a.window, a.sinks)))
                        sc[nt][j] = -INFINITY;
                }
            }
            // the row's maximum is only raised when a score passes it by 2^8: until then
            // the weights, 2^(score - m + 6), stay below fp16's 2^14
            float mx = fmaxf(fmaxf(sc[nt][0], sc[nt][1]), fmaxf(sc[nt][2], sc[nt][3]));
            if (__any_sync(0xffffffffu, mx > m[nt] + 8.0f)) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                // (a row that did not pass its own stays as it is: its bits are its own affair)
                const float mn = mx > m[nt] + 8.0f ? mx : m[nt];
                const float f = mn == m[nt] ? 1.0f : kv4_exp2(m[nt] - mn);
                m[nt] = mn;
                l[nt] *= f;
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[nt][k][j] *= f;
            }
            const float base = m[nt] == -INFINITY ? 0.0f : m[nt] - 6.0f;
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) e[j] = kv4_exp2(sc[nt][j] - base);
            l[nt] += (e[0] + e[1]) + (e[2] + e[3]);
            // the weights into B: column g is row g/2 of this tile, positions 2t, 2t+1, 2t+8, 2t+9
            const int src = 8 * t + (g >> 1);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float y0 = __shfl_sync(0xffffffffu, e[j], src), y1 = __shfl_sync(0xffffffffu, e[j], src + 4);
                const float2 hi = __half22float2(__floats2half2_rn(y0, y1));
                pb[nt][j >> 1][j & 1] = pack_half2(fmaf(hi.x, rest, y0), fmaf(hi.y, rest, y1));
            }
        }

        // outputs
        const bool cut = p0 + KD_UNIT > len || !ok0 || !ok1 || (p0 <= before && p0 + KD_UNIT > a.sinks);
        const __half2 bias_lo = bits_h2(0x64086408u);                                     // 1032
        const __half2 sixteenth = bits_h2(0x2C002C00u), bias_hi = bits_h2(0xD480D480u);   // 1/16, -72
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t *vp = unit + h * GB + 8 * HD + t * HD + g * (4 * NB), *sp = unit + h * GB + 16 * HD + 32 * NB + t * (4 * NB);
            uint32_t v[2][NB], vs[2][NB];
            lds_words<NB>(v[0], vp);
            lds_words<NB>(v[1], vp + 4 * HD);
            lds_words<NB>(vs[0], sp);
            lds_words<NB>(vs[1], sp + 4 * (4 * NB));
            if (cut) {
                // positions that no row sees may hold any bytes: their scales count as 0
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int p = p0 + 16 * h + 2 * t + 8 * j;
                    const int left = (h ? ok1 : ok0) ? len - p : 0;
                    uint32_t keep = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0x0000FFFFu : 0u;
                    if (p <= before) {
                        if (p >= a.sinks) keep &= 0xFFFF0000u;
                        if (p + 1 >= a.sinks && p < before) keep &= 0x0000FFFFu;
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) vs[j][b] &= keep;
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const __half2 d01 = bits_h2(vs[0][b]), d23 = bits_h2(vs[1][b]);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t x01 = j ? v[0][b] >> 8 : v[0][b], x23 = j ? v[1][b] >> 8 : v[1][b];
                    // 1024 + c, and 1024 + 16 c; then (c - 8) * d, every step exact
                    const __half2 a0 = __hmul2(__hsub2(bits_h2(and_or(x01, 0x000F000Fu, 0x64006400u)), bias_lo), d01);
                    const __half2 a1 = __hmul2(__hfma2(bits_h2(and_or(x01, 0x00F000F0u, 0x64006400u)), sixteenth, bias_hi), d01);
                    const __half2 a2 = __hmul2(__hsub2(bits_h2(and_or(x23, 0x000F000Fu, 0x64006400u)), bias_lo), d23);
                    const __half2 a3 = __hmul2(__hfma2(bits_h2(and_or(x23, 0x00F000F0u, 0x64006400u)), sixteenth, bias_hi), d23);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float(&c)[4] = o[nt][b * 2 + j];
                        mma_f16(c, h2bits(a0), h2bits(a1), h2bits(a2), h2bits(a3), pb[nt][h][0], pb[nt][h][1], c[0], c[1],
                                c[2], c[3]);
                    }
                }
            }
        }
        __syncwarp();                              // the stage is free
        stage ^= 1;
        p0 = pn;
        pn = p2;
        ok0 = n0;
        ok1 = n1;
    }

    cp_async_wait_all();
    __syncthreads();                               // the ring becomes the warps' results
    // ---- join the warps ----
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float sum = l[nt];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        float *pr = part[warp][nt * 4 + t];
#pragma unroll
        for (int b = 0; b < NB; b++)
            *reinterpret_cast<float4 *>(pr + b * 32 + 4 * g) =
                make_float4(o[nt][2 * b][0] + o[nt][2 * b][1], o[nt][2 * b][2] + o[nt][2 * b][3],
                            o[nt][2 * b + 1][0] + o[nt][2 * b + 1][1], o[nt][2 * b + 1][2] + o[nt][2 * b + 1][3]);
        if (g == 0) { pr[HD] = m[nt]; pr[HD + 1] = sum; }
    }
    __syncthreads();
    const int live = min(rows, R);
    for (int e = tid; e < live * HD; e += KD_THREADS) {
        const int r = e / HD, d = e - r * HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < KD_WARPS; w++) mm = fmaxf(mm, part[w][r][HD]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ov = 0.0f, lv = 0.0f;
#pragma unroll
        for (int w = 0; w < KD_WARPS; w++) {
            const float f = kv4_exp2(part[w][r][HD] - base);
            lv = fmaf(part[w][r][HD + 1], f, lv);
            ov = fmaf(part[w][r][d], f, ov);
        }
        if (!partial) {
            const int rr = chunk_row + r, tok = rr / a.group, h = kv * a.group + rr % a.group;
            T *out = (T *)a.out + (int64_t)(s.row0 + tok) * a.out_tok + h * a.out_head;
            kv_round(lv == 0.0f ? 0.0f : ov / lv, &out[d]);
        } else {
            partial[r * PS + d] = ov;
            if (d == 0) { partial[r * PS + HD] = mm; partial[r * PS + HD + 1] = lv; }
        }
    }
    if (a.parts > 1) pdl_launch_dependents();
}

// The pieces of one row of an item joined. Every warp finds the pieces' factors, then
// takes every KJ_WARPS-th piece; the warps' sums are added in order.
constexpr int KJ_WARPS = 8;
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(32 * KJ_WARPS) kv4_join_kernel(const Kv4AttnArgs a) {
    constexpr int R = 4 * NT, PS = KdLayout<HD, NT>::PS, Q = HD / 4;
    __shared__ float fac[KJ_WARPS][KD_MAX_SLOTS];
    __shared__ __align__(16) float4 part[KJ_WARPS][Q];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = blockIdx.y;
    const int ny = a.c.n_kv * a.chunks, seq = blockIdx.x / ny, y = blockIdx.x - seq * ny;
    const KdItem it = kd_item(a, seq);
    const int kv = y / a.chunks, rr = (y - kv * a.chunks) * R + r;
    const int n = (it.range.total + a.span - 1) / a.span;
    pdl_wait();
    if (rr >= it.rows || n <= 1) return;
    const Kv4Seq &s = it.s;
    auto piece = [&](int i) { return kd_partial<HD, NT>(a, blockIdx.x, i) + r * PS; };
    float mm = -INFINITY, l = 0.0f;
    for (int i = lane; i < n; i += 32) {
        fac[warp][i] = piece(i)[HD];
        mm = fmaxf(mm, fac[warp][i]);
    }
    mm = warp_max(mm);
    const float base = mm == -INFINITY ? 0.0f : mm;
    for (int i = lane; i < n; i += 32) {
        fac[warp][i] = kv4_exp2(fac[warp][i] - base);
        l = fmaf(piece(i)[HD + 1], fac[warp][i], l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncwarp();
    if (lane < Q) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int i = warp; i < n; i += KJ_WARPS) {
            const float4 p = reinterpret_cast<const float4 *>(piece(i))[lane];
            const float f = fac[warp][i];
            v.x = fmaf(p.x, f, v.x); v.y = fmaf(p.y, f, v.y); v.z = fmaf(p.z, f, v.z); v.w = fmaf(p.w, f, v.w);
        }
        part[warp][lane] = v;
    }
    __syncthreads();
    if (tid < HD) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < KJ_WARPS; w++) v += reinterpret_cast<const float *>(part[w])[tid];
        const int tok = rr / a.group, h = kv * a.group + rr - tok * a.group;
        T *out = (T *)a.out + (int64_t)(s.row0 + tok) * a.out_tok + h * a.out_head;
        kv_round(l == 0.0f ? 0.0f : v / l, &out[tid]);
    }
}

// ------------------------------------------------------------------- host ----

// Bytes of the pieces of any call with this many positions: items * parts is at most
// the number of slots wherever parts > 1. Eight rows each.
static inline size_t kv4_attention_workspace(int hd, long long max_kv) {
    return max_kv <= KD_SPAN_MIN * KD_UNIT ? 0 : (size_t)KD_MAX_SLOTS * 8 * (hd + 4) * sizeof(float);
}

template <typename T, int HD, int NT>
static int kv4_decode_launch(Kv4AttnArgs a, cudaStream_t st) {
    using L = KdLayout<HD, NT>;
    const long long rows = (long long)a.max_q * a.group;
    const long long chunks = (rows + L::R - 1) / L::R, items = (long long)a.b.n_seqs * a.c.n_kv * chunks;
    if (a.c.n_kv * chunks > 65535 || items > 0x7FFFFFFF)
        return set_err("kv4 attention: max_q %d is too large", a.max_q);
    a.chunks = (int)chunks;
    // the units that an item has at most (a window's two ends may cut a unit each)
    long long seen = a.max_kv;
    if (a.window > 0 && (long long)a.window + a.max_q + a.sinks + 2 * KD_UNIT < seen)
        seen = (long long)a.window + a.max_q + a.sinks + 2 * KD_UNIT;
    const long long units = (seen + KD_UNIT - 1) / KD_UNIT;
    // as many pieces as fill the slots once: two sequences of 40k positions take 33 us
    // so, 37 us in two rounds, 43 us in three
    long long parts = 148 * L::CTAS / items;
    if (parts > units / KD_SPAN_MIN) parts = units / KD_SPAN_MIN;
    if (parts < 1) parts = 1;
    a.span = (int)((units + parts - 1) / parts);
    if (a.span < 1) a.span = 1;
    a.parts = (int)((units + a.span - 1) / a.span);
    if (a.parts < 1) a.parts = 1;
    static std::atomic<unsigned long long> ready{0};      // devices whose limit is raised
    int dev = 0;
    CK(cudaGetDevice(&dev));
    if (dev >= 64 || !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        CK(cudaFuncSetAttribute(kv4_decode_kernel<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const dim3 grid((unsigned)a.parts, (unsigned)(a.c.n_kv * chunks), (unsigned)a.b.n_seqs);
    kv4_decode_kernel<T, HD, NT><<<grid, KD_THREADS, L::SMEM, st>>>(a);
    CK(cudaGetLastError());
    if (a.parts > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)items, (unsigned)(rows < L::R ? rows : L::R));
        cfg.blockDim = dim3(32 * KJ_WARPS);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        CK(cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, HD, NT>, a));
    }
    return 0;
}

template <typename T, int NT>
static int kv4_decode_hd(const Kv4AttnArgs &a, int hd, cudaStream_t st) {
    switch (hd) {
    case 32: return kv4_decode_launch<T, 32, NT>(a, st);
    case 64: return kv4_decode_launch<T, 64, NT>(a, st);
    default: return kv4_decode_launch<T, 128, NT>(a, st);
    }
}

}  // namespace emb
