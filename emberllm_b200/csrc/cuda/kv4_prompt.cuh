// kv4_prompt.cuh — attention over the paged 4-bit KV cache, many rows per sequence.
//
// The same mathematics as kv4_attn.cuh with tiles of 128 query rows (tokens x the query
// heads of a kv head) on tcgen05. A CTA takes RT = 2 row tiles against tiles of 128
// positions, both row tiles sharing the keys and values it unpacks (one CTA on an SM);
// where there are few rows, 1 against tiles of 64 positions (two CTAs on an SM). One
// row tile's softmax runs under the other's products. Warps have roles:
//   4 per row tile   softmax: a thread owns a row; it reads the row's scores from tensor
//        memory, raises the maximum if a score passes it by 2^8 (then O is rescaled in
//        tensor memory, which is rare), and writes the weights over the scores
//   1 per row tile   issues its products: S = Q K^T and O += P V with P from tensor
//        memory. One warp for both row tiles kept either waiting on the other's softmax,
//        a warp that unpacks as well was waited for by all (6,900 and more cycles a tile for
//        what then took 4,400; 5,300 with weights in two parts)
//   2 values, 4 (1) keys   packed codes from global memory, asked for a tile ahead, to
//        exact fp16 numbers (code - 8) * d in shared memory, swizzled as the products read
//        them; the values are transposed on the way, so both operands are K-major
// Weights and fp32 queries enter as an fp16 number and the rest (two products into
// the same sums, 22 bits); fp16 queries are exact as they are. (Weights of 11 bits for fp16
// outputs took 201 us instead of 246 for two prompts of 4k, but moved 40 % of the outputs to a
// neighbouring number: error 2.6e-4, where the outputs' own rounding is 2.0e-4.) Each
// product cuts the sum it adds to toward zero at 24 bits, two for 16 positions: sums
// are off by 2.5e-9 of themselves a position. So those of fp32 outputs leave tensor memory
// every 512 positions and are added up by rounding additions: 1.6e-6 of the outputs at any length.
// Us and error, staying / every 2048 / 1024 / 512 positions: two fp32 prompts of 4k 281, 9.9e-6 / 295,
// 5.2e-6 / 310, 2.8e-6 / 341, 1.6e-6; six ragged prompts of up to 1200 56, 1.3e-6 / 56 / 63 / 67, 9e-7
// (plain fp32 operations: 4.5e-7); 512 rows of 40,000 9.4e-5 / 5.2e-6 / 2.8e-6 / 1240 us, 1.6e-6. Those of
// fp16 outputs stay: 9.4e-5 of an output at 40,000 positions, half a step is 2.4e-4 and more.
//
// Bound by the chain scores - maximum - exponentials - weights - outputs of a row tile: tensor
// pipe 44 %, alu 40 %, exponentials 30 %, issue 50 % busy. Two prompts of 3.9-4.1k, 16 / 8 heads of
// 128, fp16: 243 us, 559 TFLOP/s; six of up to 512 rows on up to 1200 positions, fp32: 67 us. Up
// to 44 bytes are spilled and 72 loaded again a thread (fp32, heads of 32), mostly none.
#pragma once

#include <stdlib.h>

#include "kv4_attn.cuh"
#include "kv4_rule.h"

namespace emb {

constexpr int KP_ROWS = KV4_TILE_ROWS;
constexpr int KP_DRAIN = 512;             // positions whose sums stay in tensor memory (fp32)
constexpr unsigned long long KP_WAIT_NS = 1000000000ull;

// calls of ember_cuda_kv4_attention leave ERR_KV4_WAIT here, ember_cuda_kv4_status takes it
static __device__ int kv4_wait_error;

template <typename T, int HD, int RT>
struct KpLayout {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;    // fp16 parts of a query (a weight has two)
    static constexpr int NP = 64 * RT, H = NP / 64;         // positions of a tile, and its halves of 64
    static constexpr int SB = 3 - RT;                       // tiles of scores per row tile in tensor memory
    static constexpr int BUF = PARTS == 2 ? 1 : 2;          // tiles of keys and of values in shared memory
    static constexpr int PANELS = (HD + 63) / 64;           // panels of 64 fp16 (128 bytes) of a row
    static constexpr int Q_PART = PANELS * KP_ROWS * 128, Q_TILE = PARTS * Q_PART;
    static constexpr int K_PANEL = NP * 128, K_BYTES = PANELS * K_PANEL;
    static constexpr int V_PANEL = HD * 128, V_BYTES = H * V_PANEL;
    static constexpr int OFF_K = RT * Q_TILE, OFF_V = OFF_K + BUF * K_BYTES;
    static constexpr int SMEM = OFF_V + BUF * V_BYTES + 1024;   // + slack to align the base to 1024
    // tensor memory: S / P per row tile (SB tiles of NP columns: 128), then O per row tile
    static constexpr int COLS = RT * 256, COL_O = RT * 128;
    static constexpr int SOFT = 4 * RT, ISSUE = SOFT, VALS = SOFT + RT, KEYS = VALS + 2;   // first warps of the roles
    static constexpr int KEY_WARPS = RT == 2 ? 4 : 1, WARPS = RT == 2 ? 16 : 8;
    // tiles after which the sums leave tensor memory
    static constexpr int DRAIN = KP_DRAIN / NP;
    static constexpr int KN = NP / 8 / KEY_WARPS;           // positions a key thread unpacks
    static_assert(SB * NP == 128, "scores take 128 columns");
    static_assert(SMEM <= (RT == 2 ? 227 : 113) * 1024, "shared memory");
};

// what the many-row kernel takes besides (apart: 24 bytes more cost the other kernel's launch 0.6 us of
// the host)
struct KpArgs {
    Kv4AttnArgs att;
    int *err;                     // error word for waits that run out (NULL: the device's own)
    unsigned long long wait_ns;
    int lost;                     // 1: the keys' arrivals never suffice (tests of the waits)
};

template <int RT>
struct KpShared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[RT][2], p_full[RT][2], o_done[RT], o_last[RT], q_full[RT], drain;
    uint32_t tmem;
    int abort;
    uint64_t valid[4][RT];      // which positions of a tile there are, by tile number mod 4
    float rscale[RT * KP_ROWS];
};

// Wait for a phase; gives up after `ns` of waiting or as soon as another role has given up, so
// that a product that never completes ends the CTA (its rows become NaN, the error word says
// so). A poll counts as a millisecond at most: a process that the GPU was taken from for a while has not
// waited.
EMB_DEV bool kp_poll(uint32_t bar, uint32_t parity, volatile int *abort, unsigned long long ns) {
    unsigned long long t0, t1;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    while (!mbar_try_wait_at(bar, parity)) {
        if (*abort) return false;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t1));
        const unsigned long long took = min(t1 - t0, 1000000ull);
        if (took >= ns) {
            *abort = 1;
            return false;
        }
        ns -= took;
        t0 = t1;
    }
    return true;
}
// (The polling is a function of its own where two row tiles need the registers: in line in all places,
// two prompts of 4k in fp16 took 250 us instead of 241; with one row tile 512 fp32
// rows of 40,000 took 1326 apart, 1240 in line.)
static __device__ __noinline__ bool kp_poll_apart(uint32_t bar, uint32_t parity, volatile int *abort,
                                                  unsigned long long ns) {
    return kp_poll(bar, parity, abort, ns);
}
template <bool APART>
EMB_DEV bool kp_wait_ns(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned long long ns) {
    return mbar_try_wait(bar, parity) ||
           (APART ? kp_poll_apart(smem_u32(bar), parity, abort, ns) : kp_poll(smem_u32(bar), parity, abort, ns));
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
// one lane of a converged warp
EMB_DEV bool kp_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
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

// a weight's first 11 bits: an fp16 number, as long as that is a normal one (the weights that
// matter are: a row's largest is 2^6 or more). Cheaper than the rounding, which has to be widened
// again to get the rest: no spills, 281 -> 246 us for two prompts of 4k in fp16
EMB_DEV float kp_cut(float e) { return __uint_as_float(__float_as_uint(e) & 0xFFFFE000u); }

// the lower (1024 + c) and upper (1024 + 16 c) nibbles' exact (code - 8) * d
EMB_DEV uint32_t kp_low(uint32_t w, __half2 d) {
    return h2bits(__hmul2(__hsub2(bits_h2(and_or(w, 0x000F000Fu, 0x64006400u)), bits_h2(0x64086408u)), d));
}
EMB_DEV uint32_t kp_high(uint32_t w, __half2 d) {
    return h2bits(__hmul2(
        __hfma2(bits_h2(and_or(w, 0x00F000F0u, 0x64006400u)), bits_h2(0x2C002C00u), bits_h2(0xD480D480u)), d));
}

// tiles of NP positions that a CTA's rows see
template <int NP>
struct KpRange {
    int sink_tiles, lo, total;
    __device__ __forceinline__ int pos(int j) const { return (j < sink_tiles ? j : j + (lo - sink_tiles)) * NP; }
};
template <int NP>
EMB_DEV KpRange<NP> kp_range(int first_pos, int last_pos, int len, int window, int sinks) {
    KpRange<NP> r;
    const int stop = max(0, min(len, last_pos + 1)), end = (stop + NP - 1) / NP;
    const long long from = window > 0 ? (long long)first_pos - window + 1 : 0;
    r.lo = (int)max(0ll, min(from, (long long)stop)) / NP;
    r.sink_tiles = min((int)(((long long)sinks + NP - 1) / NP), r.lo);
    r.total = r.sink_tiles + end - r.lo;
    return r;
}

template <typename T, int HD, int RT>
__global__ void __launch_bounds__(32 * KpLayout<T, HD, RT>::WARPS, 3 - RT) kv4_prompt_kernel(const KpArgs args) {
    const Kv4AttnArgs &a = args.att;
    using L = KpLayout<T, HD, RT>;
    constexpr int NB = HD / 32, GB = kv4_group(HD), PARTS = L::PARTS, BUF = L::BUF, NP = L::NP, H = L::H, SB = L::SB;
    extern __shared__ uint8_t kp_raw[];
    __shared__ KpShared<RT> sh;
    const uint32_t raw = smem_u32(kp_raw);
    uint8_t *sm = kp_raw + ((1024u - (raw & 1023u)) & 1023u);
    const uint32_t sm32 = smem_u32(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kv = blockIdx.x, seq = blockIdx.y;
    const Kv4Seq s = kv4_seq(a.b, seq);
    const int rows = min(s.rows, a.max_q) * a.group;
    // the latest rows see the most positions: they go first, of all heads and sequences
    const int row_first = ((int)gridDim.z - 1 - (int)blockIdx.z) * (RT * KP_ROWS);
    if (row_first >= rows) return;
    const int row_end = min(rows, row_first + RT * KP_ROWS);
    const int pos0 = s.len - s.rows, len = min(min(s.len, a.max_kv), a.b.cap);
    const KpRange<NP> range = kp_range<NP>(pos0 + row_first / a.group, pos0 + (row_end - 1) / a.group, len, a.window, a.sinks);
    const int n = range.total;
    const int tiles = RT == 1 || row_end - row_first <= KP_ROWS ? 1 : 2;   // row tiles with rows

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.k_full[i], 32 * L::KEY_WARPS + args.lost);
            mbar_init(&sh.k_empty[i], tiles);
            mbar_init(&sh.v_full[i], 64);
            mbar_init(&sh.v_empty[i], tiles);
            for (int r = 0; r < RT; r++) { mbar_init(&sh.s_full[r][i], 1); mbar_init(&sh.p_full[r][i], KP_ROWS); }
        }
        for (int r = 0; r < RT; r++) { mbar_init(&sh.o_done[r], 1); mbar_init(&sh.o_last[r], 1); mbar_init(&sh.q_full[r], KP_ROWS); }
        mbar_init(&sh.drain, tiles);
        fence_mbar_init();
        sh.abort = 0;
    }
    if (warp == L::ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"((uint32_t)L::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    kp_fence_before();
    __syncthreads();
    kp_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int *abort = &sh.abort;
    auto kp_wait = [&](uint64_t *bar, uint32_t parity, volatile int *flag) {
        return kp_wait_ns<RT == 2>(bar, parity, flag, args.wait_ns);
    };

    if (warp < L::SOFT) {
        // ---------------------------------------------------------- softmax ----
        const int rt = warp >> 2;
        // The queries first: a warp takes 32 rows, HD / 4 lanes a row with 4 dims each.
        // Within 8 dims the order is 0,4,1,5,2,6,3,7, as the keys come out of their words:
        // neighbouring lanes exchange two numbers and store two pairs each.
        if (rt < tiles) {
            constexpr int LPR = HD / 4, RPI = 32 / LPR, BATCH = HD == 128 && sizeof(T) == 2 ? 16 : 8;
            const int sub = lane / LPR, part = lane % LPR;
            // row `lane` of the warp: where it is (there is none: the tile's first, counted as 0)
            const int mine_rr = row_first + warp * 32 + lane, my_tok = mine_rr / a.group;
            const int64_t my_off = mine_rr < rows ? (int64_t)(s.row0 + my_tok) * a.q_tok +
                                                        (kv * a.group + mine_rr - my_tok * a.group) * a.q_head
                                                  : (int64_t)s.row0 * a.q_tok + kv * a.group * a.q_head;
            const int rows_here = rows - row_first - warp * 32;
            const bool vec = !((uintptr_t)a.q % (4 * sizeof(T)) || a.q_tok % 4 || a.q_head % 4);
#pragma unroll 1
            for (int i0 = 0; i0 < 32; i0 += BATCH * RPI) {
                // all loads first, nothing between them that needs one's data
                uint32_t raw[BATCH][sizeof(T)];
#pragma unroll
                for (int e = 0; e < BATCH; e++) {
                    const int64_t off = __shfl_sync(0xffffffffu, my_off, (i0 + e * RPI + sub) & 31);
                    const T *src = (const T *)a.q + off + part * 4;
                    if (vec) {
                        lds_words<sizeof(T)>(raw[e], reinterpret_cast<const uint8_t *>(src));
                    } else if (sizeof(T) == 4) {
#pragma unroll
                        for (int k = 0; k < 4; k++) raw[e][k % sizeof(T)] = __float_as_uint(widen(src[k]));
                    } else {
                        const uint16_t *u = reinterpret_cast<const uint16_t *>(src);
                        raw[e][0] = u[0] | (uint32_t)u[1] << 16;
                        raw[e][1] = u[2] | (uint32_t)u[3] << 16;
                    }
                }
#pragma unroll
                for (int e = 0; e < BATCH; e++) {
                    const int i = i0 + e * RPI + sub;
                    float v[4];
                    if (sizeof(T) == 4) {
#pragma unroll
                        for (int k = 0; k < 4; k++) v[k] = __uint_as_float(raw[e][k % sizeof(T)]);
                    } else {
                        const float2 lo = __half22float2(bits_h2(raw[e][0])), hi = __half22float2(bits_h2(raw[e][1]));
                        v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
                    }
                    if (i >= rows_here) v[0] = v[1] = v[2] = v[3] = 0.0f;
                    // the row's largest magnitude by its bits: infinities and NaNs are larger
                    // than any number
                    uint32_t m = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) m = max(m, __float_as_uint(v[k]) & 0x7FFFFFFFu);
                    if (LPR == 32) m = __reduce_max_sync(0xffffffffu, m);
                    else
#pragma unroll
                        for (int o = LPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                    // |q| * 2^x below 2^14; the sign of the scale goes into the queries, so
                    // that a row's largest product is its largest score
                    const int x = m == 0 ? 0 : 13 - max((int)(m >> 23) - 127, -126);
                    float f1 = __int_as_float((127 + x / 2) << 23);
                    const float f2 = __int_as_float((127 + x - x / 2) << 23);
                    // (never 0: a hidden score, -inf, must stay -inf)
                    if (part == 0 && i < 32)
                        sh.rscale[warp * 32 + i] =
                            a.scale == 0.0f ? 1.0f
                                            : fmaxf(fabsf(a.scale) * KV4_LOG2E * __int_as_float((127 - x / 2) << 23) *
                                                        __int_as_float((127 - x + x / 2) << 23),
                                                    1.2e-38f);
                    if (a.scale < 0.0f) f1 = -f1;
                    if (a.scale == 0.0f) f1 = 0.0f;
                    if (m >= 0x7F800000u) f1 = __int_as_float(0x7fffffff);
                    float y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) y[k] = v[k] * f1 * f2;
                    const bool odd = part & 1;
                    const float r0 = __shfl_xor_sync(0xffffffffu, odd ? y[0] : y[2], 1);
                    const float r1 = __shfl_xor_sync(0xffffffffu, odd ? y[1] : y[3], 1);
                    // even lane: dims 0,4 and 1,5; odd lane: 2,6 and 3,7
                    const float a0 = odd ? r0 : y[0], a1 = odd ? y[2] : r0, b0 = odd ? r1 : y[1], b1 = odd ? y[3] : r1;
                    const uint32_t h0 = pack_half2(a0, a1), h1 = pack_half2(b0, b1);
                    const int c = part >> 1;
                    uint8_t *at = sm + rt * L::Q_TILE + (c >> 3) * (KP_ROWS * 128) +
                                  kp_chunk(((warp & 3) * 32 + i) & (KP_ROWS - 1), c & 7) + (odd ? 8 : 0);
                    if (i < 32) {
                        *reinterpret_cast<uint2 *>(at) = make_uint2(h0, h1);
                        if (PARTS == 2) {
                            const float2 g0 = __half22float2(bits_h2(h0)), g1 = __half22float2(bits_h2(h1));
                            *reinterpret_cast<uint2 *>(at + L::Q_PART) =
                                make_uint2(pack_half2(a0 - g0.x, a1 - g0.y), pack_half2(b0 - g1.x, b1 - g1.y));
                        }
                    }
                }
            }
        }
        kp_fence_smem();
        mbar_arrive(&sh.q_full[rt]);
        __syncwarp();
        const int r = tid, rr = row_first + r;
        const int pos = pos0 + min(rr, rows - 1) / a.group;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t col_o = mine + L::COL_O + rt * 128;
        const float rs = sh.rscale[r];
        // positions that every row of the tile sees: up to the first row's, from the last
        // row's window on
        const int first_pos = pos0 + min(row_first + rt * KP_ROWS, rows - 1) / a.group;
        const int last_pos = pos0 + (min(rows, row_first + (rt + 1) * KP_ROWS) - 1) / a.group;
        const long long all_from = a.window > 0 ? (long long)last_pos - a.window + 1 : 0;
        float m = -INFINITY, l = 0.0f, m_out = -INFINITY;
        bool ok = true;
        const int todo = rt < tiles ? n : 0;
        // The sums in tensor memory added to those of earlier tiles, which are kept in the warp's
        // own 32 rows of `out`, scaled by 2^-m_out; `last`: all of them back to tensor memory.
        // Lane r keeps its four numbers number k at place 32 k + r of the rows' numbers in a
        // row, so that the lanes' places are neighbours (in its own row, a warp's access touched 32 rows:
        // 4.9 us a time); a warp with fewer rows keeps them in its own.
        constexpr bool TAKE = sizeof(T) == 4;
        auto drain = [&](bool more, bool last) {
            constexpr int Q = HD / 4;
            const bool whole = row_first + (warp + 1) * 32 <= rows, mine_too = whole || rr < rows;
            const int row = min(rr, rows - 1), tok = row / a.group;
            const int64_t my_off = (int64_t)(s.row0 + tok) * a.out_tok + (kv * a.group + row - tok * a.group) * a.out_head;
            const bool vec = !((uintptr_t)a.out % 16 || a.out_tok % 4 || a.out_head % 4);
            // (m == m_out: nothing to scale, the addition can be left to the memory)
            const float f = m == m_out ? 1.0f : kv4_exp2(m_out - m);
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                float o[32], w[32];
                float *at[8];
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const int place = ((c + k) / 4) * 32 + lane;
                    const int64_t off = __shfl_sync(0xffffffffu, my_off, whole ? place / Q : lane);
                    at[k / 4] = reinterpret_cast<float *>(a.out) + off + (whole ? place % Q * 4 : c + k);
                    w[k] = w[k + 1] = w[k + 2] = w[k + 3] = 0.0f;
                    if (!mine_too || !more || (f == 1.0f && !last)) continue;
                    if (vec) {
                        const float4 x = __ldcg(reinterpret_cast<const float4 *>(at[k / 4]));
                        w[k] = x.x; w[k + 1] = x.y; w[k + 2] = x.z; w[k + 3] = x.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) w[k + e] = __ldcg(at[k / 4] + e);
                    }
                }
                __syncwarp();         // (the loads were some lanes', the next is the warp's)
                kp_ld32<0>(o, col_o + c);
#pragma unroll
                for (int k = 0; k < 32; k++) o[k] = fmaf(w[k], f, o[k]);
                if (last) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t u[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) u[k] = __float_as_uint(o[16 * h + k]);
                        kp_st16(col_o + c + 16 * h, u);
                    }
                } else if (mine_too) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        float *p = at[k / 4];
                        if (vec && more && f == 1.0f)
                            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(o[k]),
                                         "f"(o[k + 1]), "f"(o[k + 2]), "f"(o[k + 3])
                                         : "memory");
                        else if (vec) *reinterpret_cast<float4 *>(p) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                        else
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (more && f == 1.0f) atomicAdd(p + e, o[k + e]);
                                else p[e] = o[k + e];
                    }
                }
                __syncwarp();
            }
            if (last) kp_wait_st();
            __syncwarp();
            m_out = m;
        };
        for (int j = 0; j < todo; j++) {
            ok = kp_wait(&sh.s_full[rt][j % SB], (j / SB) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            kp_fence_after();
            // (only now: these scores followed the products of tile j - 2, so that o_done's phase
            // is told from the one before)
            const bool fresh = TAKE ? j % L::DRAIN == 0 : j == 0;      // nothing in O that counts
            if (TAKE && fresh && j > 0) {
                ok = kp_wait(&sh.o_done[rt], (j - 1) & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                kp_fence_after();
                drain(j > L::DRAIN, false);
            }
            const uint32_t at = mine + rt * 128 + (j % SB) * NP;
            float v[64];
            // a half's scores, the hidden ones -inf
            auto read = [&](int h) {
                kp_ld32<0>(v, at + h * 64);
                kp_ld32<32>(v, at + h * 64 + 32);
                const int p0 = range.pos(j) + h * 64;
                const uint64_t valid = sh.valid[j & 3][h];
                if (p0 >= all_from && p0 + 63 <= first_pos && valid == ~0ull) return;
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
            };
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int h = 0; h < H; h++) {
                read(h);
#pragma unroll
                for (int p = 0; p < 64; p++) mx[p & 3] = fmaxf(mx[p & 3], v[p]);
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * rs;
            if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                // (a row that did not pass its own stays as it is: its bits are its own affair)
                const float mn = top > m + 8.0f ? top : m;
                const float f = mn == m ? 1.0f : kv4_exp2(m - mn);
                m = mn;
                l *= f;
                if (!fresh) {
                    ok = kp_wait(&sh.o_done[rt], (j - 1) & 1, abort);    // the products into O so far
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    kp_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        kp_ld32<0>(o, col_o + c);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t u[16];
#pragma unroll
                            for (int k = 0; k < 16; k++) u[k] = __float_as_uint(o[16 * h + k] * f);
                            kp_st16(col_o + c + 16 * h, u);
                        }
                    }
                }
            }
            if (RT == 2 && tiles == 2) {
                // the row tiles take turns at the exponentials, so that one's run under the
                // other's products
                ok = rt == 0 ? j == 0 || kp_wait(&sh.p_full[RT - 1][0], (j - 1) & 1, abort)
                             : kp_wait(&sh.p_full[0][0], j & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
            const float base = m == -INFINITY ? 0.0f : m - 6.0f;
            float sum[2] = {0.0f, 0.0f};
            // the last half is still in registers; a half's weights take its scores' place,
            // first the 11 bits, then the rests
#pragma unroll 1
            for (int h = H - 1; h >= 0; h--) {
                if (h < H - 1) read(h);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const float e0 = kv4_exp2(fmaf(v[i * 32 + 2 * k], rs, -base));
                        const float e1 = kv4_exp2(fmaf(v[i * 32 + 2 * k + 1], rs, -base));
                        sum[0] += e0;
                        sum[1] += e1;
                        const float h0 = kp_cut(e0), h1 = kp_cut(e1);
                        hi[k] = pack_half2(h0, h1);
                        lo[k] = pack_half2(e0 - h0, e1 - h1);
                    }
                    kp_st16(at + h * 64 + i * 16, hi);
                    kp_st16(at + h * 64 + 32 + i * 16, lo);
                }
                kp_wait_st();
                kp_fence_before();
                mbar_arrive(&sh.p_full[rt][H == 2 ? h : j % SB]);
            }
            l += sum[0] + sum[1];
        }
        if (todo > 0 && ok) {
            // (a barrier of its own: o_done may be one or two phases behind here)
            ok = kp_wait(&sh.o_last[rt], 0, abort);
            ok = __all_sync(0xffffffffu, ok);
            kp_fence_after();
            if (TAKE && ok && todo > L::DRAIN) drain(true, true);
        }
        const bool live = rr < rows;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int tok = min(rr, rows - 1) / a.group, h = kv * a.group + min(rr, rows - 1) - tok * a.group;
        T *out = (T *)a.out + (int64_t)(s.row0 + tok) * a.out_tok + h * a.out_head;
        const bool vec = !((uintptr_t)a.out % 16 || (a.out_tok * sizeof(T)) % 16 || (a.out_head * sizeof(T)) % 16);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
            float o[32];
            if (todo > 0 && ok) kp_ld32<0>(o, col_o + c);
#pragma unroll
            for (int k = 0; k < 32; k++) o[k] = !ok ? __int_as_float(0x7fffffff) : l == 0.0f ? 0.0f : o[k] * inv;
            // (no lane may run ahead to the next, warp-wide, load)
            if (!live) {
            } else if (vec && sizeof(T) == 4) {
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
            __syncwarp();
        }
        kp_fence_before();
    } else if (warp < L::VALS) {
        // --------------------------------------------------------- products ----
        // the warp stays together and one elected lane issues
        const int rt = warp - L::ISSUE;
        if (n > 0 && rt < tiles) {
            constexpr uint32_t kind = 1u << 4 | (uint32_t)(KP_ROWS >> 4) << 24;      // fp16 x fp16 -> fp32, M = 128
            constexpr uint32_t idesc_s = kind | (uint32_t)(NP >> 3) << 17, idesc_o = kind | (uint32_t)(HD >> 3) << 17;
            const uint64_t dq = kp_desc(sm32), dk = kp_desc(sm32 + L::OFF_K), dv = kp_desc(sm32 + L::OFF_V);
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                return (bool)__all_sync(0xffffffffu, kp_wait(bar, parity, abort));
            };
            // (offsets inside shared memory are added to a descriptor's address field, in 16 bytes)
            auto outputs = [&](int j) {
                if (!wait(&sh.v_full[j % BUF], (j / BUF) & 1)) return false;
                const uint64_t v = dv + (uint32_t)(j % BUF) * (L::V_BYTES >> 4);
                const uint32_t p = tmem + rt * 128 + (j % SB) * NP, o = tmem + L::COL_O + rt * 128;
#pragma unroll
                for (int h = H - 1; h >= 0; h--) {
                    if (!wait(&sh.p_full[rt][H == 2 ? h : j % SB], (j / SB) & 1)) return false;
                    kp_fence_after();
                    if (kp_elect()) {
#pragma unroll
                        for (int q = 0; q < 2; q++)
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                kp_mma_ts(o, p + h * 64 + q * 32 + k * 8, v + ((h * L::V_PANEL + k * 32) >> 4), idesc_o,
                                          (sizeof(T) == 4 ? j % L::DRAIN : j) > 0 || h < H - 1 || q + k > 0);
                        if (h == 0) {
                            kp_commit(&sh.o_done[rt]);
                            kp_commit(&sh.v_empty[j % BUF]);
                            if (j == n - 1) kp_commit(&sh.o_last[rt]);
                        }
                    }
                    __syncwarp();
                }
                return true;
            };
            auto scores = [&](int j) {
                // the weights that tile j - SB left where these scores go have been used
                if (!wait(&sh.k_full[j % BUF], (j / BUF) & 1) ||
                    (j >= SB && !wait(&sh.o_done[rt], (j - SB) & 1)))
                    return false;
                kp_fence_after();
                const uint64_t k0 = dk + (uint32_t)(j % BUF) * (L::K_BYTES >> 4);
                const uint32_t d = tmem + rt * 128 + (j % SB) * NP;
                const uint64_t q0 = dq + (uint32_t)rt * (L::Q_TILE >> 4);
                // (the rests first: each product's sum is cut to fp32, while it is small here)
                if (kp_elect()) {
#pragma unroll
                    for (int q = PARTS - 1; q >= 0; q--)
#pragma unroll
                        for (int k = 0; k < HD / 16; k++)
                            kp_mma_ss(d, q0 + ((q * L::Q_PART + (k >> 2) * (KP_ROWS * 128) + (k & 3) * 32) >> 4),
                                      k0 + (((k >> 2) * L::K_PANEL + (k & 3) * 32) >> 4), idesc_s, q < PARTS - 1 || k > 0);
                    kp_commit(&sh.s_full[rt][j % SB]);
                    kp_commit(&sh.k_empty[j % BUF]);
                }
                __syncwarp();
                return true;
            };
            // SB scores ahead; with one tile of scores, the next follow the outputs, while the
            // other row tile's softmax runs
            bool ok = wait(&sh.q_full[rt], 0);
            for (int j = 0; ok && j < SB && j < n; j++) ok = scores(j);
            for (int j = 0; ok && j < n; j++) {
                ok = outputs(j);
                if (ok && j + SB < n) ok = scores(j + SB);
            }
            // products in flight end before tensor memory is given back
            int never = 0;
            if (kp_elect()) kp_commit(&sh.drain);
            __syncwarp();
            kp_wait_ns<RT == 2>(&sh.drain, 0, &never, KP_WAIT_NS);
        }
    } else if (warp < L::KEYS + L::KEY_WARPS) {
        // ------------------------------------------------- keys and values ----
        // A tile's packed words are loaded while the tile before is made operands, and
        // the numbers of its pages a tile before that. Where there is no page, page 0 is
        // read: its positions count as hidden, its values' scales as 0.
        const bool keys = warp >= L::KEYS;
        const int ps = 1 << a.c.page_shift;
        const int32_t *table = a.b.table + (size_t)seq * a.b.table_stride;
        const uint8_t *base = a.c.data + (size_t)kv * a.c.chunk;
        const uint64_t stride = (uint64_t)a.c.n_kv * a.c.chunk;
        auto page_at = [&](int j, int in_tile) {
            const int p = range.pos(j) + in_tile;
            return j < n && p < len ? __ldg(table + (p >> a.c.page_shift)) : -1;
        };
        auto group = [&](int page, int p) {
            const bool is = (unsigned)page < (unsigned)a.c.n_pages;
            return base + (is ? (uint64_t)(uint32_t)page * stride + ((p & (ps - 1)) >> 4) * GB : 0);
        };
        if (keys) {
            // thread: word column t of the positions first + 8 i + low
            constexpr int KN = L::KN;
            const int t = lane >> 3, low = lane & 7, first = (warp - L::KEYS) * (8 * KN);
            struct Packed {
                uint32_t w[KN][NB], d[KN][NB < 2 ? 1 : NB / 2];
                uint64_t ok;              // which of the positions there are
            };
            static_assert(KN == 8 || KN == 4, "a warp's positions are 32 or 64 bits of the mask");
            int pg[(KN + 1) / 2];
            auto pages = [&](int j) {
#pragma unroll
                for (int i = 0; i < KN; i += 2) pg[i / 2] = page_at(j, first + 8 * i);
            };
            auto load = [&](Packed &u, int j) {
                const int p0 = range.pos(j);
                u.ok = 0;
                if (j >= n) return;
#pragma unroll
                for (int i = 0; i < KN; i++) {
                    const int p = first + i * 8 + low, r = p & 15;
                    const uint8_t *g = group(pg[i / 2], p0 + p);
                    lds_words<NB>(u.w[i], g + r * (HD / 2) + t * (4 * NB));
                    lds_words<NB / 2>(u.d[i], g + 16 * HD + r * (2 * NB));
                    if (p0 + p < len && (unsigned)pg[i / 2] < (unsigned)a.c.n_pages) u.ok |= 1ull << (i * 8 + low);
                }
            };
            auto make = [&](const Packed &u, int j) {
                // which of the warp's positions there are, for the softmax
                const uint32_t ok0 = __reduce_or_sync(0xffffffffu, (uint32_t)u.ok);
                const uint32_t ok1 = KN == 8 ? __reduce_or_sync(0xffffffffu, (uint32_t)(u.ok >> 32)) : 0;
                if (!__all_sync(0xffffffffu, j < BUF || kp_wait(&sh.k_empty[j % BUF], ((j / BUF) + 1) & 1, abort)))
                    return false;
                uint8_t *dst = sm + L::OFF_K + (j % BUF) * L::K_BYTES;
                if (lane == 0) {
                    if (KN == 8) sh.valid[j & 3][warp - L::KEYS] = (uint64_t)ok1 << 32 | ok0;
                    else reinterpret_cast<uint32_t *>(sh.valid[j & 3])[warp - L::KEYS] = ok0;
                }
#pragma unroll
                for (int i = 0; i < KN; i++) {
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const __half2 dd = bits_h2(__byte_perm(u.d[i][b / 2], 0, (b & 1) ? 0x3232 : 0x1010));
                        const uint32_t x = u.w[i][b], y = x >> 8;
                        const uint4 q = make_uint4(kp_low(x, dd), kp_high(x, dd), kp_low(y, dd), kp_high(y, dd));
                        *reinterpret_cast<uint4 *>(dst + (b >> 1) * L::K_PANEL +
                                                   kp_chunk(first + i * 8 + low, 4 * (b & 1) + t)) = q;
                    }
                }
                kp_fence_smem();
                mbar_arrive(&sh.k_full[j % BUF]);
                return true;
            };
            Packed ua, ub;
            pages(0);
            load(ua, 0);
            pages(1);
            for (int j = 0; j < n; j += 2) {
                load(ub, j + 1);
                pages(j + 2);
                if (!make(ua, j)) break;
                if (j + 1 >= n) break;
                load(ua, j + 2);
                pages(j + 3);
                if (!make(ub, j + 1)) break;
            }
        } else {
            // thread: value words g of the 8 positions 8 c .. of a half; item i is half
            // i % H of tile i / H
            const int t64 = tid - 32 * L::VALS, c = t64 & 7, g = t64 >> 3;
            struct Packed { uint32_t w[4][NB], d[4][NB]; };
            int pg;
            auto page = [&](int i) { pg = page_at(i / H, (i % H) * 64 + 8 * c); };
            const int before = kv4_before(pos0 + row_first / a.group, a.window);
            auto load = [&](Packed &u, int i) {
                if (i >= n * H) return;
                const int p0 = range.pos(i / H) + (i % H) * 64;
                const uint8_t *gr = group(pg, p0 + 8 * c);
                const bool is = (unsigned)pg < (unsigned)a.c.n_pages;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int pair = (c & 1) * 4 + e;
                    lds_words<NB>(u.w[e], gr + 8 * HD + pair * HD + g * (4 * NB));
                    lds_words<NB>(u.d[e], gr + 16 * HD + 32 * NB + pair * (4 * NB));
                }
                // positions that no row sees may hold any bytes: their scales count as 0
                if (!is || p0 + 64 > len || (p0 <= before && p0 + 64 > a.sinks)) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int p = p0 + 8 * c + 2 * e;
                        auto seen = [&](int q) { return is && q < len && (q < a.sinks || q > before); };
                        const uint32_t keep = (seen(p) ? 0xFFFFu : 0u) | (seen(p + 1) ? 0xFFFF0000u : 0u);
#pragma unroll
                        for (int b = 0; b < NB; b++) u.d[e][b] &= keep;
                    }
                }
            };
            auto make = [&](const Packed &u, int i) {
                const int j = i / H;
                if (i % H == 0 &&
                    !__all_sync(0xffffffffu, j < BUF || kp_wait(&sh.v_empty[j % BUF], ((j / BUF) + 1) & 1, abort)))
                    return false;
                uint8_t *dst = sm + L::OFF_V + (j % BUF) * L::V_BYTES + (i % H) * L::V_PANEL;
#pragma unroll
                for (int b = 0; b < NB; b++) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t w = k < 2 ? u.w[e][b] : u.w[e][b] >> 8;
                            x[e] = (k & 1) ? kp_high(w, bits_h2(u.d[e][b])) : kp_low(w, bits_h2(u.d[e][b]));
                        }
                        *reinterpret_cast<uint4 *>(dst + kp_chunk(b * 32 + 4 * g + k, c)) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                if (i % H == H - 1) {
                    kp_fence_smem();
                    mbar_arrive(&sh.v_full[j % BUF]);
                }
                return true;
            };
            Packed ua, ub;
            page(0);
            load(ua, 0);
            page(1);
            for (int i = 0; i < n * H; i += 2) {
                load(ub, i + 1);
                page(i + 2);
                if (!make(ua, i)) break;
                if (i + 1 >= n * H) break;
                load(ua, i + 2);
                page(i + 3);
                if (!make(ub, i + 1)) break;
            }
        }
    }
    __syncwarp();
    __syncthreads();
    kp_fence_after();
    if (tid == 0 && *abort) atomicExch(args.err ? args.err : &kv4_wait_error, ERR_KV4_WAIT);
    if (warp == L::ISSUE)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::COLS) : "memory");
}

// ------------------------------------------------------------------- host ----

template <typename T, int HD, int RT>
static int kv4_prompt_launch(const Kv4AttnArgs &a, int *err, cudaStream_t st) {
    // tests: keys that never arrive, and so many us until the waits for them run out
    const char *us = getenv("EMBER_KV4_LOST_KEYS_US");
    const KpArgs args = { a, err, us ? strtoull(us, nullptr, 10) * 1000ull : KP_WAIT_NS, us != nullptr };
    using L = KpLayout<T, HD, RT>;
    static std::atomic<unsigned long long> ready{0};      // devices whose limit is raised
    int dev = 0;
    CK(cudaGetDevice(&dev));
    if (dev >= 64 || !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        CK(cudaFuncSetAttribute(kv4_prompt_kernel<T, HD, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const long long tiles = ((long long)a.max_q * a.group + RT * KP_ROWS - 1) / (RT * KP_ROWS);
    if (tiles > 65535) return set_err("kv4 attention: max_q %d is too large", a.max_q);
    const dim3 grid((unsigned)a.c.n_kv, (unsigned)a.b.n_seqs, (unsigned)tiles);
    kv4_prompt_kernel<T, HD, RT><<<grid, 32 * L::WARPS, L::SMEM, st>>>(args);
    CK(cudaGetLastError());
    return 0;
}

template <typename T, int RT>
static int kv4_prompt_hd(const Kv4AttnArgs &a, int hd, int *err, cudaStream_t st) {
    switch (hd) {
    case 32: return kv4_prompt_launch<T, 32, sizeof(T) == 2 ? 1 : RT>(a, err, st);    // (fp16: one row tile always)
    case 64: return kv4_prompt_launch<T, 64, RT>(a, err, st);
    default: return kv4_prompt_launch<T, 128, RT>(a, err, st);
    }
}

}  // namespace emb
