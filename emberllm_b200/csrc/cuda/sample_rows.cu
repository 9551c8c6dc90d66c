// sample_rows.cu — one draw per row of a batch of logits.
//
// The tokens of a row are ordered by (logit descending, index ascending); each
// has the weight w = exp((logit - max) / temperature), rounded to a multiple of
// 2^-44 and held as an integer. Every truncation keeps a prefix of that order, so
// the kept weight is the smallest of the prefixes' weights, and the draw is again
// a prefix: the first token whose running weight reaches floor(u * kept) + 1. All
// of them ask one question -- where does a running sum (of weights or of ones)
// reach a target. It is answered without sorting: the distances max - logit are
// binned, the bins' sums added up, and the bin in which the target lies is binned
// again (by the bits of the logit, then by index) until its tokens fit a list;
// there each token adds up the weights before it. The sums are integers: no order of
// additions can change a token.
//
// A cluster of CTAs holds the row in shared memory, so the logits are read once;
// they exchange maxima, bins and lists through distributed shared memory: each adds up
// its own bins by groups of 32, and who looks for a target reads the groups, then the
// bins of one group, of all. Bound by instructions, 97 a token and lane at half of the
// issue slots: the weight (11 double-precision operations: the draw compares sums of
// up to 393,216 weights, and a token next to a border must not change), its bin and
// the atomic additions; memory would take 48 us of the 413 us for 512 rows of 151,936
// (64 rows with truncations 76 us, one of 32,000 12 us with the call). With the running
// sums over all bins in every CTA it took 454 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "ember_kv4.h"
#include "runtime_internal.cuh"

namespace cg = cooperative_groups;

namespace emb {

constexpr int SR_THREADS = 512, SR_WARPS = SR_THREADS / 32;
constexpr int SR_BINS = 1024;
constexpr int SR_LIST = 768;              // tokens of a bin that are compared one by one
constexpr int SR_MAX_CLUSTER = 8;
static_assert(SR_BINS == 32 * 32, "32 groups of 32 bins");

typedef unsigned long long u64;

constexpr int SR_SUB = SR_THREADS;        // finer bins of the listed tokens
constexpr int SR_FEW = 64;                // listed tokens compared with each other at once

// One CTA's shared memory; the row's slice of logits follows.
struct SrShared {
    struct {
        u64 w[SR_BINS];                   // this CTA's bins: weights ...
        uint32_t c[SR_BINS];              // ... and, where top_k needs them, tokens
    } bin;
    struct {
        u64 w[32];
        uint32_t c[32];
    } group;                              // sums of 32 bins each
    struct {
        u64 key[SR_LIST], w[SR_LIST];     // the first CTA: tokens of the bin that is looked through
    } list;
    u64 run_w[32];                        // running sums over the row's groups
    uint32_t run_c[32];
    u64 sub_w[SR_SUB];                    // the first CTA: sums of the finer bins
    uint32_t sub_c[SR_SUB];
    int few[SR_LIST];                     // tokens of one of them
    double pow2[64];                      // 2^(j/64)
    u64 part_w[SR_WARPS], sum_w;          // block sums; the CTA's weight within min_p
    uint32_t part_c[SR_WARPS];
    float part_hi[SR_WARPS], part_lo[SR_WARPS], hi, lo;
    int part_i[SR_WARPS], hi_i;
    int list_n[2], few_n;
    u64 at_w, at_c;                       // running sums before a bin that is looked through
    uint32_t to_c;                        // tokens up to its end
    u64 res_key, res_w;                   // a search's result
    int bin_at;
};

EMB_DEV float sr_logit(float v) { return v != v ? -INFINITY : v; }

// 2^(y/64) for -3000 < y <= 0 (the weights' limit is 31.25 / ln 2 * 64 = 2885): 2^(k/64) from the table, k the nearest integer, times
// exp(f * ln2/64), |f| <= 1/2, by its Taylor polynomial of degree 4 (the next term is
// below 4e-14, a weight's rounding 2.8e-14). 11 double-precision operations; the
// library's exp takes some 30.
EMB_DEV double sr_exp2_64(double y, const double *pow2) {
    constexpr double C = 0.69314718055994530942 / 64.0;
    const double t = y + 6755399441055744.0;                 // 1.5 * 2^52: the nearest integer
    const int k = (int)__double_as_longlong(t);
    const double f = y - (t - 6755399441055744.0);
    double q = C * C * C * C / 24.0;
    q = __fma_rn(q, f, C * C * C / 6.0);
    q = __fma_rn(q, f, C * C / 2.0);
    q = __fma_rn(q, f, C);
    q = __fma_rn(q, f, 1.0);
    q *= pow2[k & 63];
    return __longlong_as_double(__double_as_longlong(q) + ((long long)(k >> 6) << 52));
}

// Ascending keys are descending logits; -0 counts as +0. Key 0x80000000, that of -0,
// is no token's.
constexpr uint32_t SR_LAST_KEY = 0xFF800000u;   // -inf
EMB_DEV uint32_t sr_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u >> 31) ? u : 0x7FFFFFFFu - u;
}
EMB_DEV float sr_key_logit(uint32_t k) { return __uint_as_float((k >> 31) ? k : 0x7FFFFFFFu - k); }

struct SrRow {
    float mx, limit;                      // distances above limit weigh nothing: w < 2^-45
    double slope;                         // -64 / (temperature * ln 2)
};
// The weight comes from the logits in double precision: their difference in fp32 is
// rounded, which moved weights by 1e-7 and merged neighbouring logits.
EMB_DEV double sr_weight(const SrRow &r, float l, const double *pow2) {
    return r.mx - l > r.limit ? 0.0 : sr_exp2_64(((double)r.mx - (double)l) * r.slope, pow2);
}
// w is in [0, 1]: adding 2^52 to w * 2^44 leaves the integer in the mantissa
EMB_DEV u64 sr_units(double w) {
    return (u64)__double_as_longlong(__fma_rn(w, 17592186044416.0, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// 64-bit addition in shared memory by 32-bit atomics: whoever makes the lower word
// wrap carries into the upper one
EMB_DEV void sr_add(u64 *at, u64 v) {
    uint32_t *p = reinterpret_cast<uint32_t *>(at);
    const uint32_t lo = (uint32_t)v, old = atomicAdd(p, lo);
    const uint32_t hi = (uint32_t)(v >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(p + 1, hi);
}

// Level 0 bins: proportional to the distance, so a bin's tokens are neighbours in the
// order; the last bin holds what is farther than the scale's reach (also inf * 0).
EMB_DEV int sr_bin(float scale, float d) { return (int)fminf(d * scale, (float)(SR_BINS - 1)); }

// The smallest key whose distance lies in bin `at` or a later one, by a whole warp:
// 32 candidates at a time.
EMB_DEV uint32_t sr_bin_start(float mx, float scale, int at, int lane) {
    uint32_t k0 = sr_key(mx), k1 = SR_LAST_KEY;     // k0 before it (or it, at = 0); k1 in it or later
    if (at == 0) return k0;
    while (k1 - k0 > 1) {
        const uint32_t step = (k1 - k0 + 32) / 33;
        const uint32_t k = min((unsigned long long)k1, k0 + (unsigned long long)step * (lane + 1));
        const unsigned in = __ballot_sync(~0u, sr_bin(scale, mx - sr_key_logit(k)) >= at);
        const int first = in ? __ffs(in) - 1 : 32;
        if (first < 32) k1 = __shfl_sync(~0u, k, first);
        if (first > 0) k0 = __shfl_sync(~0u, k, first - 1);
    }
    return k1;
}

// The smallest distance in bin `at` or a later one, by a whole warp: d * scale is rounded
// once, so it is next to at / scale.
EMB_DEV float sr_bin_distance(float scale, int at, int lane) {
    if (at == 0) return 0.0f;
    const float d = __uint_as_float(__float_as_uint((float)at / scale) - 16 + lane);
    const unsigned in = __ballot_sync(~0u, sr_bin(scale, d) >= at);
    return __shfl_sync(~0u, d, in ? __ffs(in) - 1 : 31);
}

// where a running sum reaches its target
struct SrFound {
    u64 key;                              // (logit's key, index): ascending in the order
    u64 w;                                // running weight there, inclusive
};

template <typename T>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_rows_kernel(EmberSampleRows a, int slice, bool vec) {
    extern __shared__ __align__(16) uint8_t sr_raw[];
    SrShared &sh = *reinterpret_cast<SrShared *>(sr_raw);
    float *val = reinterpret_cast<float *>(sr_raw + (sizeof(SrShared) + 15) / 16 * 16);   // the slice's logits
    cg::cluster_group cl = cg::this_cluster();
    const int nc = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x / nc;
    const int i0 = min(a.vocab, rank * slice), n = min(a.vocab, i0 + slice) - i0;
    const T *x = (const T *)a.logits + (int64_t)row * a.stride + i0;
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
    const int top_k = a.top_k ? a.top_k[row] : 0;

    // ---- what the row needs (while its logits are on their way) ----
    if (tid < 2) sh.list_n[tid] = 0;
    if (tid < 64) sh.pow2[tid] = exp2((double)tid / 64.0);
    for (int b = tid; b < SR_BINS; b += SR_THREADS) { sh.bin.w[b] = 0; sh.bin.c[b] = 0; }
    SrRow R;
    R.slope = -64.0 / 0.69314718055994530942 / (double)temp;
    R.limit = (float)fmin(31.25 * (double)temp, 3.4e38);   // exp(-31.25) < 2^-45
    const bool use_k = top_k > 0 && top_k < a.vocab, use_p = top_p > 0.0f && top_p < 1.0f,
               use_min = min_p > 0.0f && min_p < 1.0f;
    const bool need_total = use_p || !(use_k || use_min);
    float weigh_to = R.limit;             // distances up to which weights are needed
    if (use_min && !need_total)           // (with a margin for the rounding of this bound)
        weigh_to = fminf(weigh_to, (float)fmin(-log((double)min_p) * (double)temp * 1.0001 + 1e-30, 3.4e38));

    // ---- the slice into shared memory; the row's maximum (first index) and minimum ----
    float hi = -INFINITY, lo = INFINITY;
    int hi_i = 0x7FFFFFFF;
    auto take = [&](float v, int i) {
        if (v > hi || (v == hi && i < hi_i)) { hi = v; hi_i = i; }
    };
    constexpr int W = 16 / sizeof(T);
    auto see = [&](float v, int i) {
        v = sr_logit(v);
        val[i] = v;
        if (v > hi) { hi = v; hi_i = i0 + i; }
        if (v > -INFINITY) lo = fminf(lo, v);
    };
    const int nv = vec ? n / W : 0;
#pragma unroll 4
    for (int j = tid; j < nv; j += SR_THREADS) {
        const uint4 q = __ldg(reinterpret_cast<const uint4 *>(x) + j);
        const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
        for (int k = 0; k < W; k++) see(widen(e[k]), j * W + k);
    }
    for (int i = nv * W + tid; i < n; i += SR_THREADS) see(widen(x[i]), i);
    auto warp_take = [&]() {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            take(__shfl_xor_sync(~0u, hi, o), __shfl_xor_sync(~0u, hi_i, o));
            lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
        }
    };
    warp_take();
    if (lane == 0) { sh.part_hi[warp] = hi; sh.part_lo[warp] = lo; sh.part_i[warp] = hi_i; }
    __syncthreads();
    hi = lane < SR_WARPS ? sh.part_hi[lane] : -INFINITY;
    lo = lane < SR_WARPS ? sh.part_lo[lane] : INFINITY;
    hi_i = lane < SR_WARPS ? sh.part_i[lane] : 0x7FFFFFFF;
    warp_take();
    if (nc > 1) {
        if (tid == 0) { sh.hi = hi; sh.lo = lo; sh.hi_i = hi_i; }
        cl.sync();
        const SrShared *o = cl.map_shared_rank(&sh, min(lane, nc - 1));
        hi = o->hi;
        lo = o->lo;
        hi_i = o->hi_i;
        warp_take();
    }
    const bool greedy = !(temp > 0.0f) || hi == -INFINITY;
    if (greedy) {
        if (rank == 0 && tid == 0) a.out[row] = hi == -INFINITY ? 0 : hi_i;
        if (nc > 1) cl.sync();            // no CTA leaves while its maximum may be read
        return;
    }

    // an infinite maximum: the infinite logits weigh 1, the others nothing, as 0 and -inf do
    const int n4 = n / 4;
    float4 *val4 = reinterpret_cast<float4 *>(val);
    if (hi == INFINITY) {
        for (int i = tid; i < n; i += SR_THREADS) val[i] = val[i] == INFINITY ? 0.0f : -INFINITY;
        hi = lo = 0.0f;
        __syncthreads();
    }
    R.mx = hi;
    // f(logit, index) for every token of the slice, four at a time
    auto each = [&](auto f) {
        for (int i = tid; i < n4; i += SR_THREADS) {
            const float4 v = val4[i];
            f(v.x, i0 + 4 * i); f(v.y, i0 + 4 * i + 1); f(v.z, i0 + 4 * i + 2); f(v.w, i0 + 4 * i + 3);
        }
        for (int i = 4 * n4 + tid; i < n; i += SR_THREADS) f(val[i], i0 + i);
    };
    auto sync = [&]() {
        if (nc > 1) cl.sync();
        else __syncthreads();
    };
    const float far = lo == INFINITY ? 0.0f : R.mx - lo;    // of the finite logits (inf if that overflows)

    // ---- bins ----
    auto binning = [&](float to) { return fminf((float)(SR_BINS - 2) / fmaxf(to, 1e-30f), 3.0e38f); };
    auto clear = [&]() {
        sync();                           // nobody reads the bins or the list any more
        for (int b = tid; b < SR_BINS; b += SR_THREADS) { sh.bin.w[b] = 0; sh.bin.c[b] = 0; }
        __syncthreads();
    };
    auto add = [&](int b, u64 w) {
        if (use_k) atomicAdd(&sh.bin.c[b], 1u);
        if (w) sr_add(&sh.bin.w[b], w);
    };
    // running sums over a warp's lanes
    auto warp_run = [&](u64 &w, uint32_t &c) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 vw = __shfl_up_sync(~0u, w, o);
            const uint32_t vc = __shfl_up_sync(~0u, c, o);
            if (lane >= o) { w += vw; c += vc; }
        }
    };
    // adds the sums of the earlier warps (part_*)
    auto before = [&](u64 &w, uint32_t &c) {
        u64 pw = lane < warp ? sh.part_w[lane] : 0;
        uint32_t pc = lane < warp ? sh.part_c[lane] : 0;
#pragma unroll
        for (int o = SR_WARPS / 2; o; o >>= 1) {
            pw += __shfl_xor_sync(~0u, pw, o);
            pc += __shfl_xor_sync(~0u, pc, o);
        }
        w += __shfl_sync(~0u, pw, 0);
        c += __shfl_sync(~0u, pc, 0);
    };
    // the bins' groups of 32 and the row's running sums over them, the same in every CTA
    auto merge = [&]() {
        __syncthreads();
        for (int g = warp; g < 32; g += SR_WARPS) {
            u64 w = sh.bin.w[32 * g + lane];
            uint32_t c = use_k ? sh.bin.c[32 * g + lane] : 0;
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                w += __shfl_xor_sync(~0u, w, o);
                c += __shfl_xor_sync(~0u, c, o);
            }
            if (lane == 0) { sh.group.w[g] = w; sh.group.c[g] = c; }
        }
        sync();
        if (warp == 0) {
            u64 w = 0;
            uint32_t c = 0;
#pragma unroll
            for (int q = 0; q < SR_MAX_CLUSTER; q++)
                if (q < nc) {
                    const SrShared *o = cl.map_shared_rank(&sh, q);
                    w += o->group.w[lane];
                    c += o->group.c[lane];
                }
            warp_run(w, c);
            sh.run_w[lane] = w;
            sh.run_c[lane] = c;
        }
        __syncthreads();
    };

    // the whole row, its weights where the row needs them
    float top = binning(use_k ? far : fminf(far, weigh_to));
    bool top_valid = false, clean = true;
    u64 in_min = 0;                       // this thread's weight within min_p
    auto bin_row = [&](bool weights) {
        if (!clean) clear();              // the first time the bins are zeros
        clean = false;
        in_min = 0;
        if (need_total) {
            // every token has its weight, one beyond the limit 0: no branch but those that
            // all lanes take alike. The additions of four tokens come after their weights:
            // an atomic between them would hold back the next one's table entry, and the
            // upper words need what the lower ones returned.
            const double mx = (double)R.mx;
            auto weigh = [&](float l, int &b) {
                const float d = R.mx - l;
                const bool on = d <= R.limit;
                const double e = sr_exp2_64((mx - (double)(on ? l : R.mx)) * R.slope, sh.pow2);
                const u64 w = on ? sr_units(e) : 0;
                b = sr_bin(top, d);
                if (use_min && e >= (double)min_p) in_min += w;
                return w;
            };
            for (int i = tid; i < n4; i += SR_THREADS) {
                const float4 v = val4[i];
                int b[4];
                const u64 w[4] = {weigh(v.x, b[0]), weigh(v.y, b[1]), weigh(v.z, b[2]), weigh(v.w, b[3])};
                uint32_t old[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (use_k) atomicAdd(&sh.bin.c[b[k]], 1u);
                    old[k] = atomicAdd(reinterpret_cast<uint32_t *>(&sh.bin.w[b[k]]), (uint32_t)w[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t up = (uint32_t)(w[k] >> 32) + (old[k] + (uint32_t)w[k] < old[k] ? 1u : 0u);
                    if (up) atomicAdd(reinterpret_cast<uint32_t *>(&sh.bin.w[b[k]]) + 1, up);
                }
            }
            for (int i = 4 * n4 + tid; i < n; i += SR_THREADS) {
                int b;
                const u64 w = weigh(val[i], b);
                if (use_k) atomicAdd(&sh.bin.c[b], 1u);
                sr_add(&sh.bin.w[b], w);
            }
        } else {
            each([&](float l, int) {
                const float d = R.mx - l;
                u64 w = 0;
                if (weights && d <= weigh_to) {
                    const double e = sr_weight(R, l, sh.pow2);
                    w = sr_units(e);
                    if (use_min && e >= (double)min_p) in_min += w;
                }
                add(sr_bin(top, d), w);
            });
        }
        merge();
        top_valid = true;
    };
    // the bin in which the running sum, before_* at the first one's start, reaches the
    // target (the last bin, should it reach it nowhere): its group, then the bin in it;
    // before_* become the sums at its start
    auto bin_at = [&](u64 target, bool count, u64 &before_w, u64 &before_c) {
        if (warp == 0) {
            unsigned in = __ballot_sync(~0u, (count ? before_c + sh.run_c[lane] : before_w + sh.run_w[lane]) >= target);
            const int g = in ? __ffs(in) - 1 : 31;
            u64 w0 = 0, w;
            uint32_t c0 = 0, c;
#pragma unroll
            for (int q = 0; q < SR_MAX_CLUSTER; q++)
                if (q < nc) {
                    const SrShared *o = cl.map_shared_rank(&sh, q);
                    w0 += o->bin.w[32 * g + lane];
                    c0 += use_k ? o->bin.c[32 * g + lane] : 0;
                }
            w = w0;
            c = c0;
            warp_run(w, c);
            const u64 bw = before_w + (g ? sh.run_w[g - 1] : 0) + w, bc = before_c + (g ? sh.run_c[g - 1] : 0) + c;
            in = __ballot_sync(~0u, (count ? bc : bw) >= target);
            if (lane == (in ? __ffs(in) - 1 : 31)) {
                sh.bin_at = 32 * g + lane;
                sh.at_w = bw - w0;
                sh.at_c = bc - c0;
                sh.to_c = (uint32_t)bc;
            }
        }
        __syncthreads();
        before_w = sh.at_w;
        before_c = sh.at_c;
        return sh.bin_at;
    };
    // the distances in a bin of level 0
    auto bin_distances = [&](int at, float &d0, float &d1) {
        d0 = sr_bin_distance(top, at, lane);
        d1 = INFINITY;
        if (at < SR_BINS - 1) d1 = __uint_as_float(__float_as_uint(sr_bin_distance(top, at + 1, lane)) - 1);
    };
    // tokens with base - logit in [d0, d1] and an index in [j0, j1] to the
    // first CTA's list; their number, list_n, may be more than the list holds
    int turn = 0;
    auto gather = [&](float base, float d0, float d1, int j0, int j1) {
        // (the list's place was last read before a sync that all have passed; so was the
        // other counter, which is made ready for the next time)
        SrShared *first = cl.map_shared_rank(&sh, 0);
        if (rank == 0 && tid == 0) sh.list_n[turn ^ 1] = 0;
        auto push = [&](float l, int i) {
            if (i < j0 || i > j1) return;
            const int e = atomicAdd(&first->list_n[turn], 1);
            if (e < SR_LIST) {
                first->list.key[e] = ((u64)sr_key(l) << 32) | (uint32_t)i;
                first->list.w[e] = sr_units(sr_weight(R, l, sh.pow2));
            }
        };
        for (int i = tid; i < n4; i += SR_THREADS) {
            float4 v = val4[i];
            v.x = base - v.x; v.y = base - v.y; v.z = base - v.z; v.w = base - v.w;
            int in = (v.x >= d0 && v.x <= d1) | (v.y >= d0 && v.y <= d1) << 1 | (v.z >= d0 && v.z <= d1) << 2 |
                     (v.w >= d0 && v.w <= d1) << 3;
            for (; in; in &= in - 1) {    // mostly none
                const int e = __ffs(in) - 1;
                push(val[4 * i + e], i0 + 4 * i + e);
            }
        }
        for (int i = 4 * n4 + tid; i < n; i += SR_THREADS)
            if (base - val[i] >= d0 && base - val[i] <= d1) push(val[i], i0 + i);
        sync();
        turn ^= 1;
    };
    // in the first CTA: which of the list's tokens takes the running sum to target; all
    // CTAs learn its key and the running weight
    auto resolve = [&](int tokens, u64 target, bool count, u64 before_w, u64 before_c, float base, float d0, float d1,
                       bool ties, bool last) {
        int m = tokens;
        if (tokens > SR_FEW) {
            // finer bins, by distance or, among equal logits, by index (a product of zero and
            // infinity, d1's, goes to the last bin)
            const float sub = (float)SR_SUB / (d1 - d0);
            int shift = 0;
            while (((uint32_t)(a.vocab - 1) >> shift) >= SR_SUB) shift++;
            auto sub_of = [&](u64 key) {
                const float d = base - sr_key_logit((uint32_t)(key >> 32));
                return ties ? (int)((uint32_t)key >> shift) : (int)fminf((d - d0) * sub, (float)(SR_SUB - 1));
            };
            sh.sub_w[tid] = 0;
            sh.sub_c[tid] = 0;
            if (tid == 0) sh.few_n = 0;
            __syncthreads();
            for (int i = tid; i < tokens; i += SR_THREADS) {
                const int b = sub_of(sh.list.key[i]);
                atomicAdd(&sh.sub_c[b], 1u);
                sr_add(&sh.sub_w[b], sh.list.w[i]);
            }
            __syncthreads();
            const u64 mw = sh.sub_w[tid];
            const uint32_t mc = sh.sub_c[tid];
            u64 w = mw;
            uint32_t c = mc;
            warp_run(w, c);
            if (lane == 31) { sh.part_w[warp] = w; sh.part_c[warp] = c; }
            __syncthreads();
            before(w, c);
            const u64 s = count ? before_c + c : before_w + w, s0 = count ? s - mc : s - mw;
            if (s0 < target && s >= target) {
                sh.bin_at = tid;
                sh.at_w = before_w + w - mw;
                sh.at_c = before_c + c - mc;
            }
            __syncthreads();
            for (int i = tid; i < tokens; i += SR_THREADS)
                if (sub_of(sh.list.key[i]) == sh.bin_at) sh.few[atomicAdd(&sh.few_n, 1)] = i;
            __syncthreads();
            m = sh.few_n;
            before_w = sh.at_w;
            before_c = sh.at_c;
        } else {
            if (tid < tokens) sh.few[tid] = tid;
            __syncthreads();
        }
        for (int e = tid; e < m; e += SR_THREADS) {
            const int i = sh.few[e];
            const u64 key = sh.list.key[i];
            u64 w = before_w, c = before_c;
            for (int j = 0; j < m; j++)
                if (sh.list.key[sh.few[j]] < key) { w += sh.list.w[sh.few[j]]; c++; }
            const u64 s0 = count ? c : w, s = count ? c + 1 : w + sh.list.w[i];
            if (s0 < target && s >= target)
                for (int q = 0; q < (last ? 1 : nc); q++) {
                    SrShared *o = cl.map_shared_rank(&sh, q);
                    o->res_key = key;
                    o->res_w = w + sh.list.w[i];
                }
        }
    };
    // the first place in the order where the running sum reaches target; the last search's
    // result is the first CTA's alone, the others are done
    auto find = [&](u64 target, bool count, bool last) {
        u64 before_w = 0, before_c = 0;
        // the part of the row that is binned: level 0, all by distance; 1, keys in
        // [k0, k1]; 2, one key, by index. Each level's bin is a 1/512 of its range at most,
        // so there are at most 4 of keys and 3 of indices.
        uint32_t k0 = 0, k1 = SR_LAST_KEY;
        int level = 0, shift = 0, j0 = 0, j1 = 0x7FFFFFFF;
        for (;;) {
            const int at = bin_at(target, count, before_w, before_c);
            float base = 0.0f, d0, d1;
            if (level == 0) {
                base = R.mx;
                bin_distances(at, d0, d1);
            } else {
                if (level == 1) {
                    k1 = (uint32_t)min((long long)k1, k0 + ((at + 1ll) << shift) - 1);
                    k0 += (uint32_t)at << shift;
                } else {
                    j1 = min((long long)j1, j0 + ((at + 1ll) << shift) - 1);
                    j0 += at << shift;
                }
                // (as numbers, -0 would let +0 in)
                d0 = 0.0f - sr_key_logit(k0 == 0x80000000u ? 0x80000001u : k0);
                d1 = 0.0f - sr_key_logit(k1);
            }
            gather(base, d0, d1, j0, j1);
            const int tokens = cl.map_shared_rank(&sh, 0)->list_n[turn ^ 1];
            if (tokens <= SR_LIST) {
                if (last) sync();         // all have read the number: they may leave
                if (rank == 0) resolve(tokens, target, count, before_w, before_c, base, d0, d1, level && k0 == k1, last);
                if (!last) sync();
                else __syncthreads();
                return SrFound{sh.res_key, sh.res_w};
            }
            if (level == 0) {
                k0 = sr_bin_start(R.mx, top, at, lane);
                k1 = at < SR_BINS - 1 ? sr_bin_start(R.mx, top, at + 1, lane) - 1 : SR_LAST_KEY;
            }
            if (k0 == k1 && level != 2) { j0 = 0; j1 = a.vocab - 1; }
            level = k0 == k1 ? 2 : 1;
            const uint32_t width = level == 1 ? k1 - k0 : (uint32_t)(j1 - j0);
            shift = 0;
            while ((width >> shift) >= SR_BINS) shift++;
            clear();
            each([&](float l, int i) {
                const uint32_t k = sr_key(l);
                if (k >= k0 && k <= k1 && i >= j0 && i <= j1)
                    add((int)((level == 1 ? k - k0 : (uint32_t)(i - j0)) >> shift), sr_units(sr_weight(R, l, sh.pow2)));
            });
            merge();
            top_valid = false;
        }
    };

    // ---- the searches: the last of the k where no total is needed, then top_p, top_k
    // and the draw (one loop, so that the search is in the code once) ----
    u64 kept = ~0ull;
    for (int stage = 0; stage < 4; stage++) {
        if ((stage == 0 && (!use_k || need_total)) || (stage == 1 && !use_p) || (stage == 2 && !use_k)) continue;
        if (!top_valid) bin_row(stage > 0);
        u64 target = (u64)top_k;
        if (stage == 0) {
            // no weights beyond the last of the k: binned by tokens alone
            u64 w = 0, c = 0;
            float d0, d1;
            bin_distances(bin_at(target, true, w, c), d0, d1);
            const int tokens = (int)sh.to_c;
            if (tokens <= SR_LIST) {
                // they and the rest of their bin fit the list: the first CTA does the rest
                gather(R.mx, 0.0f, d1, 0, 0x7FFFFFFF);
                if (rank != 0) return;
                constexpr int Q = (SR_LIST + SR_THREADS - 1) / SR_THREADS;
                u64 mine[Q], sum = 0;
#pragma unroll
                for (int q = 0; q < Q; q++) {
                    const int i = q * SR_THREADS + tid;
                    mine[q] = ~0ull;
                    if (i >= tokens) continue;
                    const u64 key = sh.list.key[i];
                    u64 w = 0;
                    int c = 0;
                    for (int j = 0; j < tokens; j++)
                        if (sh.list.key[j] < key) { w += sh.list.w[j]; c++; }
                    if (c >= top_k) continue;
                    mine[q] = w;
                    if (!use_min || sr_weight(R, sr_key_logit((uint32_t)(key >> 32)), sh.pow2) >= (double)min_p)
                        sum += sh.list.w[i];
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
                if (lane == 0) sh.part_w[warp] = sum;
                __syncthreads();
                sum = 0;
                for (int k = 0; k < SR_WARPS; k++) sum += sh.part_w[k];
                const u64 r = min((u64)((u > 0.0f ? (double)fminf(u, 1.0f) : 0.0) * (double)sum), sum - 1);
#pragma unroll
                for (int q = 0; q < Q; q++) {
                    const int i = min(q * SR_THREADS + tid, SR_LIST - 1);
                    if (mine[q] <= r && r < mine[q] + sh.list.w[i]) a.out[row] = (int)(sh.list.key[i] & 0xFFFFFFFFu);
                }
                return;
            }
        } else if (stage == 1) {
            const u64 total = sh.run_w[31];
            target = max(1ull, min((u64)ceil((double)top_p * (double)total), total));
        } else if (stage == 3) {
            kept = min(kept, sh.run_w[31]);
            if (use_min) {
                // the weight of what min_p keeps, over the cluster
#pragma unroll
                for (int o = 16; o; o >>= 1) in_min += __shfl_xor_sync(~0u, in_min, o);
                if (lane == 0) sh.part_w[warp] = in_min;
                __syncthreads();
                if (tid == 0) {
                    u64 w = 0;
                    for (int k = 0; k < SR_WARPS; k++) w += sh.part_w[k];
                    sh.sum_w = w;
                }
                sync();
                u64 w = 0;
                for (int q = 0; q < nc; q++) w += cl.map_shared_rank(&sh, q)->sum_w;
                kept = min(kept, w);
            }
            target = min((u64)((u > 0.0f ? (double)fminf(u, 1.0f) : 0.0) * (double)kept), kept - 1) + 1;
        }
        const SrFound f = find(target, stage == 0 || stage == 2, stage == 3);
        if (stage == 0) {
            weigh_to = fminf(weigh_to, R.mx - sr_key_logit((uint32_t)(f.key >> 32)));
            top = binning(weigh_to);
            top_valid = false;
        } else if (stage < 3) {
            kept = min(kept, f.w);
        } else if (rank == 0 && tid == 0) {
            a.out[row] = (int)(f.key & 0xFFFFFFFFu);
        }
    }
}

// logits of a CTA that shares an SM (228 KB, 1 KB of them the system's per CTA) with another
constexpr int SR_SLICE_OF_TWO = (int)((228 * 1024 / 2 - 1024 - (sizeof(SrShared) + 15) / 16 * 16) / 4 / 8 * 8);
static_assert(SR_SLICE_OF_TWO == 20040, "the rule's comment names it");

template <typename T>
static int sample_rows_launch(const EmberSampleRows &a, int n_sm, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    // As few CTAs a row as hold it with two of them on an SM, more while SMs are idle. Us for 512 /
    // 148 rows, one CTA an SM and two: 20,480 tokens 68 / 23 and 66 / 23, 40,960 138 / 44 and 133 / 48,
    // 81,920 315 / 96 and 294 / 92. Above 8 x 20,040 tokens there is no choice: 430 at 160,000, 691 at
    // 163,840.
    int nc = 1;
    while (nc < SR_MAX_CLUSTER && (a.vocab + nc - 1) / nc > SR_SLICE_OF_TWO) nc *= 2;
    while (nc < SR_MAX_CLUSTER && (long long)a.n_rows * nc * 2 <= n_sm && a.vocab / (nc * 2) >= 2048) nc *= 2;
    const int slice = (a.vocab + nc * W - 1) / (nc * W) * W;
    const size_t smem = (sizeof(SrShared) + 15) / 16 * 16 + (size_t)slice * 4;
    const bool vec = !((uintptr_t)a.logits % 16 || (a.stride * (int64_t)sizeof(T)) % 16);
    int dev = 0;
    CK(cudaGetDevice(&dev));
    static std::atomic<unsigned long long> ready{0};      // devices whose limit is raised
    if (dev >= 64 || !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        const size_t most = (sizeof(SrShared) + 15) / 16 * 16 + (size_t)EMBER_SAMPLE_MAX_VOCAB / SR_MAX_CLUSTER * 4;
        CK(cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    if ((long long)a.n_rows * nc > 0x7FFFFFFFll) return set_err("sample rows: too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_rows * nc));
    cfg.blockDim = dim3(SR_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)nc;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CK(cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, a, slice, vec));
    return 0;
}

}  // namespace emb

using namespace emb;

extern "C" int ember_cuda_sample_rows(const EmberSampleRows *args, void *stream) {
    const char *who = "sample rows";
    if (!args) return set_err("%s: null arguments", who);
    const EmberSampleRows &a = *args;
    if (a.dtype != EMBER_DT_F32 && a.dtype != EMBER_DT_F16)
        return set_err("%s: dtype %d is not EMBER_DT_F32 or EMBER_DT_F16", who, a.dtype);
    if (a.n_rows < 0) return set_err("%s: negative n_rows", who);
    if (a.vocab < 1 || a.vocab > EMBER_SAMPLE_MAX_VOCAB)
        return set_err("%s: vocab %d is outside [1, %d]", who, a.vocab, EMBER_SAMPLE_MAX_VOCAB);
    if (a.n_rows == 0) return 0;
    if (a.stride < 0) return set_err("%s: negative stride", who);
    const size_t es = a.dtype == EMBER_DT_F32 ? 4 : 2;
    if ((uintptr_t)a.logits % es) return set_err("%s: logits are not aligned to their type", who);
    int dev = -1;
    const void *need[3] = {a.logits, a.u, a.out}, *opt[4] = {a.temperature, a.top_p, a.min_p, a.top_k};
    for (int i = 0; i < 7; i++) {
        const void *p = i < 3 ? need[i] : opt[i - 3];
        if (i >= 3 && !p) continue;
        cudaPointerAttributes attr;
        if (!p || cudaPointerGetAttributes(&attr, p) != cudaSuccess ||
            (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged)) {
            cudaGetLastError();
            return set_err("%s: logits, u, out and the settings must be device memory", who);
        }
        if (i == 0) dev = attr.device;
        else if (attr.device != dev) return set_err("%s: the arrays belong to different devices", who);
        if ((uintptr_t)p % 4 && i) return set_err("%s: the settings, u and out must be 4-byte aligned", who);
    }
    int prev = -1;
    CK(cudaGetDevice(&prev));
    if (prev != dev) CK(cudaSetDevice(dev));
    cudaStream_t st = (cudaStream_t)stream;
    const int rc = a.dtype == EMBER_DT_F32 ? sample_rows_launch<float>(a, 148, st) : sample_rows_launch<__half>(a, 148, st);
    if (prev != dev) cudaSetDevice(prev);
    return rc;
}
