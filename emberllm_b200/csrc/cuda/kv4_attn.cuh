// kv4_attn.cuh — attention over the paged 4-bit KV cache, few rows per sequence.
//
// Per row at position pos and per query head: s_p = scale * (q . k_p) over the
// visible positions p, weights exp(s_p - m) with m the largest visible s_p, and
// out = sum weights_p * v_p / sum weights_p, in one pass over the cache: when a
// larger score appears, what was summed so far is multiplied by exp(m_old - m_new).
//
// Bound by memory (144 bytes a position and kv head of 128) once the codes are
// turned into matrix operands cheaply enough: at 44 bytes per ns and SM there are
// about 3 lane instructions per element. So the codes go from global memory to
// registers in the order of the fragments of mma m16n8k16 and are made operands
// there: shared memory would be written and read 4x the packed bytes. tcgen05
// takes its operands from shared memory and at least 64 rows of one side; with a
// handful of query rows per kv head it has nothing to gain here (prompts use it).
//   scores   A = keys (16 positions x 16 dims): a nibble of a word, masked in
//            place, IS an fp16 subnormal (code * 2^-24, or code * 2^-20 for the
//            upper nibbles, whose query elements carry 1/16), so 5 instructions
//            make 8 operands; B = queries. Sums per 32-block, to which the block's
//            scale and -8 * (sum of the queries) are applied in fp32.
//   outputs  A = values (16 dims x 16 positions), made exact fp16 numbers
//            (code - 8) * d; B = the weights, times 2^14.
// Queries and weights take two columns of B each, the fp16 rounding and the
// rounded rest: 22 bits for the price of idle columns. A query row is first scaled
// by a power of two so that its largest element is below 2^14.
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
    int splits, chunks;           // cache splits per sequence; row chunks per kv head
    float *ws;
};

constexpr int KD_WARPS = 4;
constexpr int KD_THREADS = 32 * KD_WARPS;
constexpr int KD_UNIT = 16;        // positions a warp takes at a time (within one page)
constexpr float KV4_LOG2E = 1.44269504088896341f;

EMB_DEV bool kv4_visible(int pos, int p, int window, int sinks) {
    return p <= pos && (window == 0 || pos - p < window || p < sinks);
}

EMB_DEV float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// C += A (16x16) * B (16x8), fp16 operands, fp32 sums
EMB_DEV void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

EMB_DEV uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
EMB_DEV __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
EMB_DEV uint32_t pack_half2(float lo, float hi) { return h2bits(__floats2half2_rn(lo, hi)); }
// {v & mask, or magic}: one lop3
EMB_DEV uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic) { return (v & mask) | magic; }

// W consecutive 32-bit words (or one 16-bit piece, W = 0) without polluting L1
template <int W>
EMB_DEV void ldg_words(uint32_t (&r)[W < 1 ? 1 : W], const void *p) {
    if (W == 0) r[0] = __ldg(reinterpret_cast<const unsigned short *>(p));
    else if (W == 1) r[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    else if (W == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        r[0] = v.x; r[W - 1] = v.y;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        r[0] = v.x; r[1 % W] = v.y; r[2 % W] = v.z; r[W - 1] = v.w;
    }
}

// what a lane loads of one unit of 16 positions: key words of positions g and g+8,
// value bytes of positions 2t, 2t+1, 2t+8, 2t+9, and those positions' scales
template <int HD>
struct KdUnit {
    static constexpr int NB = HD / 32;
    static constexpr int VW = NB / 2;                 // words of a lane's value bytes (0: 16 bits)
    static constexpr int VR = VW < 1 ? 1 : VW;
    uint32_t k[2][NB], ks[2][VR], v[4][VR], vs[4][VR];
};

template <int HD>
EMB_DEV void kd_load(KdUnit<HD> &u, const uint8_t *chunk, int slot0, int ps, int lane) {
    constexpr int NB = HD / 32;
    const int g = lane >> 2, t = lane & 3;
    const uint8_t *k = chunk + (size_t)(slot0 + g) * (HD / 2) + t * (4 * NB);
    const uint8_t *ks = chunk + (size_t)ps * HD + (slot0 + g) * (2 * NB);
    ldg_words<NB>(u.k[0], k);
    ldg_words<NB>(u.k[1], k + 8 * (HD / 2));
    ldg_words<KdUnit<HD>::VW>(u.ks[0], ks);
    ldg_words<KdUnit<HD>::VW>(u.ks[1], ks + 8 * (2 * NB));
    const uint8_t *v = chunk + (size_t)ps * (HD / 2) + (size_t)(slot0 + 2 * t) * (HD / 2) + g * (2 * NB);
    const uint8_t *vs = chunk + (size_t)ps * HD + ps * (2 * NB) + (slot0 + 2 * t) * (2 * NB);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int o = (j & 1) + (j >> 1) * 8;
        ldg_words<KdUnit<HD>::VW>(u.v[j], v + o * (HD / 2));
        ldg_words<KdUnit<HD>::VW>(u.vs[j], vs + o * (2 * NB));
    }
}

// the units of KD_UNIT positions a sequence's rows see: those of the sinks, then
// those from the first row's window on
struct KdRange {
    int sink_units, lo, total;
    __device__ __forceinline__ int unit(int i) const { return i < sink_units ? i : lo + (i - sink_units); }
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

// NT column tiles of 4 query rows each. Grid: (split, kv head * row chunk, sequence).
// A row's partial result: max (log2 units), sum, HD outputs, in units of 2^14.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(KD_THREADS) kv4_decode_kernel(const Kv4AttnArgs a) {
    constexpr int NB = HD / 32, R = 4 * NT, PS = HD + 4;   // PS: row stride of partials, in floats
    __shared__ __align__(16) uint4 qf[NT][NB][32];
    __shared__ float xs8[R][NB], rscale[R];
    __shared__ __align__(16) float part[KD_WARPS][R][PS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kv = blockIdx.y / a.chunks, chunk_row = (blockIdx.y - kv * a.chunks) * R;
    const Kv4Seq s = kv4_seq(a.b, blockIdx.z);
    const int rows = min(s.rows, a.max_q) * a.group - chunk_row;   // rows of this chunk (token-major, head in group)
    if (rows <= 0) return;
    const int pos0 = s.len - s.rows;                       // position of the sequence's first row
    const int len = min(min(s.len, a.max_kv), a.b.cap);
    const KdRange range = kd_range(pos0 + chunk_row / a.group, pos0 + (chunk_row + min(rows, R) - 1) / a.group, len,
                                   a.window, a.sinks);
    const int u0 = (int)((long long)range.total * blockIdx.x / a.splits),
              u1 = (int)((long long)range.total * (blockIdx.x + 1) / a.splits);

    // ---- queries into B fragments ----
    {
        float *x = &part[0][0][0];                         // [R][HD] scaled queries
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int r = warp * NT + i, rr = chunk_row + r;
            float v[NB], m = 0.0f;
            bool finite = true;
            const int tok = rr / a.group, h = kv * a.group + rr % a.group;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                v[b] = 0.0f;
                if (r < rows)
                    v[b] = widen(((const T *)a.q)[(int64_t)(s.row0 + tok) * a.q_tok + h * a.q_head + b * 32 + lane]);
                finite = finite && fabsf(v[b]) < INFINITY;
                m = fmaxf(m, fabsf(v[b]));
            }
            m = warp_max(m);
            finite = __all_sync(0xffffffffu, finite);
            // 2^e with m * 2^e in [2^13, 2^14), in two factors that are normal numbers
            const int e = m > 0.0f ? 13 - ilogbf(m) : 0;
            const float f1 = __int_as_float((127 + e / 2) << 23), f2 = __int_as_float((127 + e - e / 2) << 23);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float y = finite ? v[b] * f1 * f2 : __int_as_float(0x7fffffff);
                const __half hi = __float2half_rn(y);
                const __half lo = __float2half_rn(y - __half2float(hi));
                float sum = __half2float(hi) + __half2float(lo);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                x[r * HD + b * 32 + lane] = y;
                if (lane == 0) xs8[r][b] = 8.0f * sum;
            }
            if (lane == 0) rscale[r] = a.scale * KV4_LOG2E / f1 / f2;
        }
        __syncthreads();
        for (int f = warp; f < NT * NB; f += KD_WARPS) {
            // column g: row nt*4 + g/2, its fp16 rounding (even g) or the rest (odd g)
            const float *xr = x + (f / NB * 4 + (g >> 1)) * HD + (f % NB) * 32 + 8 * t;
            float y[8];
#pragma unroll
            for (int n = 0; n < 8; n++) {
                y[n] = xr[n] * ((n & 1) ? 0.0625f : 1.0f);
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
    const int ps = 1 << a.c.page_shift;
    auto page_of = [&](int i) { return i < u1 ? kv4_page(a.c, a.b, blockIdx.z, range.unit(i) * KD_UNIT) : -1; };

    KdUnit<HD> nxt;
    int i = u0 + warp;
    int page = page_of(i), page_next = page_of(i + KD_WARPS);
    if (page >= 0) kd_load<HD>(nxt, kv4_chunk_ptr(a.c, page, kv), (range.unit(i) * KD_UNIT) & (ps - 1), ps, lane);
    for (; i < u1; i += KD_WARPS) {
        const KdUnit<HD> cur = nxt;
        const bool have = page >= 0;
        page = page_next;
        page_next = page_of(i + 2 * KD_WARPS);
        if (page >= 0)
            kd_load<HD>(nxt, kv4_chunk_ptr(a.c, page, kv), (range.unit(i + KD_WARPS) * KD_UNIT) & (ps - 1), ps, lane);
        if (!have) continue;
        const int p0 = range.unit(i) * KD_UNIT;

        // scores of positions p0 + g and p0 + g + 8 for row nt*4 + t
        float sc[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) sc[nt][0] = sc[nt][1] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t w0 = cur.k[0][b], w1 = cur.k[1][b];
            const uint32_t h0 = w0 >> 8, h1 = w1 >> 8;
            const float d0 = __half2float((b & 1) ? __high2half(bits_h2(cur.ks[0][b / 2])) : __low2half(bits_h2(cur.ks[0][b / 2])));
            const float d1 = __half2float((b & 1) ? __high2half(bits_h2(cur.ks[1][b / 2])) : __low2half(bits_h2(cur.ks[1][b / 2])));
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint4 f = qf[nt][b][lane];
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_f16(c, w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, f.x, f.y);
                mma_f16(c, h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, f.z, f.w);
                const float e8 = xs8[nt * 4 + t][b];
                sc[nt][0] = fmaf(d0, fmaf(c[0] + c[1], 16777216.0f, -e8), sc[nt][0]);
                sc[nt][1] = fmaf(d1, fmaf(c[2] + c[3], 16777216.0f, -e8), sc[nt][1]);
            }
        }

        // softmax: the row's lanes are those of equal t
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 4 + t;
            const int pos = pos0 + (chunk_row + r) / a.group;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int p = p0 + g + 8 * j;
                const bool see = p < len && kv4_visible(pos, p, a.window, a.sinks);
                sc[nt][j] = see ? sc[nt][j] * rscale[r] : -INFINITY;
            }
            float mx = fmaxf(sc[nt][0], sc[nt][1]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (__any_sync(0xffffffffu, mx > m[nt])) {
                const float mn = fmaxf(m[nt], mx);
                const float f = m[nt] == -INFINITY ? 0.0f : kv4_exp2(m[nt] - mn);
                m[nt] = mn;
                l[nt] *= f;
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[nt][k][j] *= f;
            }
            const float base = m[nt] == -INFINITY ? 0.0f : m[nt] - 14.0f;
            const float e0 = kv4_exp2(sc[nt][0] - base), e1 = kv4_exp2(sc[nt][1] - base);
            l[nt] += e0 + e1;
            // the weights into B: column g is row g/2 of this tile, positions 2t, 2t+1, 2t+8, 2t+9
            const int src = 8 * t + (g >> 1);
            float y[4];
            y[0] = __shfl_sync(0xffffffffu, e0, src);
            y[1] = __shfl_sync(0xffffffffu, e0, src + 4);
            y[2] = __shfl_sync(0xffffffffu, e1, src);
            y[3] = __shfl_sync(0xffffffffu, e1, src + 4);
            pb[nt][0] = pack_half2(y[0], y[1]);
            pb[nt][1] = pack_half2(y[2], y[3]);
            if (g & 1) {
                const float2 h0 = __half22float2(bits_h2(pb[nt][0])), h1 = __half22float2(bits_h2(pb[nt][1]));
                pb[nt][0] = pack_half2(y[0] - h0.x, y[1] - h0.y);
                pb[nt][1] = pack_half2(y[2] - h1.x, y[3] - h1.y);
            }
        }

        // outputs. Positions behind the length may hold any bytes: their scales count as 0
        uint32_t vs[4][KdUnit<HD>::VR];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool in = p0 + 2 * t + (j & 1) + (j >> 1) * 8 < len;
#pragma unroll
            for (int k = 0; k < KdUnit<HD>::VR; k++) vs[j][k] = in ? cur.vs[j][k] : 0u;
        }
        const __half2 bias_lo = bits_h2(0x64086408u);                        // 1032
        const __half2 sixteenth = bits_h2(0x2C002C00u), bias_hi = bits_h2(0xD480D480u);   // 1/16, -72
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t sel = (b & 1) ? 0x7632u : 0x5410u;
            const __half2 d01 = bits_h2(__byte_perm(vs[0][b / 2], vs[1][b / 2], sel));
            const __half2 d23 = bits_h2(__byte_perm(vs[2][b / 2], vs[3][b / 2], sel));
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int byte = 2 * (b & 1) + j;
                const uint32_t bs = byte | (byte << 4) | ((4 + byte) << 8) | ((4 + byte) << 12);
                const uint32_t x01 = __byte_perm(cur.v[0][b / 2], cur.v[1][b / 2], bs);
                const uint32_t x23 = __byte_perm(cur.v[2][b / 2], cur.v[3][b / 2], bs);
                // 1024 + c, and 1024 + 16 c; then (c - 8) * d, every step exact
                const __half2 a0 = __hmul2(__hsub2(bits_h2(and_or(x01, 0x000F000Fu, 0x64006400u)), bias_lo), d01);
                const __half2 a1 = __hmul2(__hfma2(bits_h2(and_or(x01, 0x00F000F0u, 0x64006400u)), sixteenth, bias_hi), d01);
                const __half2 a2 = __hmul2(__hsub2(bits_h2(and_or(x23, 0x000F000Fu, 0x64006400u)), bias_lo), d23);
                const __half2 a3 = __hmul2(__hfma2(bits_h2(and_or(x23, 0x00F000F0u, 0x64006400u)), sixteenth, bias_hi), d23);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    mma_f16(o[nt][b * 2 + j], h2bits(a0), h2bits(a1), h2bits(a2), h2bits(a3), pb[nt][0], pb[nt][1]);
            }
        }
    }

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
    float *ws = a.ws + (((size_t)blockIdx.z * gridDim.y + blockIdx.y) * a.splits + blockIdx.x) * (R * PS);
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
        if (a.splits == 1) {
            const int rr = chunk_row + r, tok = rr / a.group, h = kv * a.group + rr % a.group;
            T *out = (T *)a.out + (int64_t)(s.row0 + tok) * a.out_tok + h * a.out_head;
            kv_round(lv == 0.0f ? 0.0f : ov / lv, &out[d]);
        } else {
            ws[r * PS + d] = ov;
            if (d == 0) { ws[r * PS + HD] = mm; ws[r * PS + HD + 1] = lv; }
        }
    }
    if (a.splits > 1) pdl_launch_dependents();
}

// The splits' partial results of one (kv head, row chunk, sequence) joined.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(KD_THREADS) kv4_join_kernel(const Kv4AttnArgs a) {
    constexpr int R = 4 * NT, PS = HD + 4;
    const int kv = blockIdx.x / a.chunks, chunk_row = (blockIdx.x - kv * a.chunks) * R;
    const Kv4Seq s = kv4_seq(a.b, blockIdx.y);
    const int rows = min(min(s.rows, a.max_q) * a.group - chunk_row, R);
    pdl_wait();
    const float *ws = a.ws + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * a.splits * (R * PS);
    for (int e = threadIdx.x; e < rows * HD; e += KD_THREADS) {
        const int r = e / HD, d = e - r * HD;
        float mm = -INFINITY;
        for (int i = 0; i < a.splits; i++) mm = fmaxf(mm, ws[(size_t)i * R * PS + r * PS + HD]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ov = 0.0f, lv = 0.0f;
        for (int i = 0; i < a.splits; i++) {
            const float *p = ws + (size_t)i * R * PS + r * PS;
            const float f = kv4_exp2(p[HD] - base);
            lv = fmaf(p[HD + 1], f, lv);
            ov = fmaf(p[d], f, ov);
        }
        const int rr = chunk_row + r, tok = rr / a.group, h = kv * a.group + rr % a.group;
        T *out = (T *)a.out + (int64_t)(s.row0 + tok) * a.out_tok + h * a.out_head;
        kv_round(lv == 0.0f ? 0.0f : ov / lv, &out[d]);
    }
}

// ------------------------------------------------------------------- host ----

struct Kv4Plan {
    int nt, chunks, splits;
};

constexpr int KD_WANT = 148 * 6;   // CTAs to aim at when the cache is split

static inline long long kd_most_splits(long long positions) {
    return (positions + KD_UNIT - 1) / KD_UNIT / (2 * KD_WARPS);   // two units a warp at least
}

static inline Kv4Plan kv4_plan(const Kv4AttnArgs &a) {
    Kv4Plan p;
    const long long rows = (long long)a.max_q * a.group;
    p.nt = rows <= 4 ? 1 : 2;
    p.chunks = (int)((rows + 4 * p.nt - 1) / (4 * p.nt));
    const long long base = (long long)a.b.n_seqs * a.c.n_kv * p.chunks;
    long long seen = a.max_kv;
    if (a.window > 0 && (long long)a.window + a.max_q + a.sinks < seen) seen = (long long)a.window + a.max_q + a.sinks;
    long long splits = (KD_WANT + base - 1) / base;
    if (splits > kd_most_splits(seen)) splits = kd_most_splits(seen);
    p.splits = splits < 1 ? 1 : (int)splits;
    return p;
}

// Bytes of the partial results of any split call with this many positions: the
// CTAs of a split call number fewer than 2 * KD_WANT, with at most 8 rows each.
static inline size_t kv4_attention_workspace(int hd, long long max_kv) {
    return kd_most_splits(max_kv) < 2 ? 0 : (size_t)2 * KD_WANT * 8 * (hd + 4) * 4;
}

template <typename T, int HD, int NT>
static int kv4_decode_launch(const Kv4AttnArgs &a, int n_kv, cudaStream_t st) {
    const dim3 grid((unsigned)a.splits, (unsigned)(n_kv * a.chunks), (unsigned)a.b.n_seqs);
    kv4_decode_kernel<T, HD, NT><<<grid, KD_THREADS, 0, st>>>(a);
    CK(cudaGetLastError());
    if (a.splits > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(n_kv * a.chunks), (unsigned)a.b.n_seqs);
        cfg.blockDim = dim3(KD_THREADS);
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
    case 32: return kv4_decode_launch<T, 32, NT>(a, a.c.n_kv, st);
    case 64: return kv4_decode_launch<T, 64, NT>(a, a.c.n_kv, st);
    default: return kv4_decode_launch<T, 128, NT>(a, a.c.n_kv, st);
    }
}

template <typename T>
static int kv4_attention_launch(Kv4AttnArgs a, int hd, cudaStream_t st) {
    const Kv4Plan p = kv4_plan(a);
    if ((long long)a.c.n_kv * p.chunks > 65535) return set_err("kv4 attention: max_q %d is too large", a.max_q);
    a.splits = p.splits;
    a.chunks = p.chunks;
    return p.nt == 1 ? kv4_decode_hd<T, 1>(a, hd, st) : kv4_decode_hd<T, 2>(a, hd, st);
}

}  // namespace emb
