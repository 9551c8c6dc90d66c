// kv4.cu — the paged 4-bit KV cache: store, read, and the host side of the
// attention over it (kernels in kv4_attn.cuh for few rows
// per sequence and kv4_prompt.cuh for many).
#include <cuda_runtime.h>

#include <math.h>

#include "kv4.cuh"
#include "kv4_prompt.cuh"
#include "kv4_rule.h"
#include "runtime_internal.cuh"

namespace emb {

struct Kv4Io {
    void *k, *v;
    int64_t k_tok, k_head, v_tok, v_head;
};

EMB_DEV void load8(const float *p, bool vec, float (&x)[8]) {
    if (vec) {
        const float4 f = reinterpret_cast<const float4 *>(p)[0], g = reinterpret_cast<const float4 *>(p)[1];
        x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
        x[4] = g.x; x[5] = g.y; x[6] = g.z; x[7] = g.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = p[j];
    }
}
EMB_DEV void load8(const __half *p, bool vec, float (&x)[8]) {
    if (vec) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const __half2 *h = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = __half22float2(h[j]);
            x[2 * j] = f.x; x[2 * j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __half2float(p[j]);
    }
}

// code of x for scale d: floor(x / d + 8.5) in exact arithmetic, clamped; y = x * inv,
// inv = 1 / d, is off by less than 2e-6. Adding 1.5 * 2^23 + 8 rounds y + 8 to the nearest
// whole number, in the lower bits. Within 1e-4 of a border (c - 8.5) that may be the
// wrong side: a border times d has 13 significant bits, exact in fp32, so comparing x
// with it settles it. (No conversion instructions: their pipe takes 16 lanes a cycle.)
EMB_DEV uint32_t kv4_code(float x, float d, float inv) {
    const float y = fminf(fmaxf(__fmul_rn(x, inv), -9.0f), 9.0f);
    const float r = __fadd_rn(y, 12582920.0f);
    int c = (int)(__float_as_uint(r) & 0xFFu);                   // -1 (0xFF) .. 17
    c = c == 0xFF ? -1 : c;
    const float whole = __fadd_rn(r, -12582912.0f);
    if (fabsf(__fadd_rn(y, 8.0f) - whole) > 0.4999f) {
        const float ax = d < 0.0f ? -x : x, ad = fabsf(d);
        if (ax < __fmul_rn(whole - 8.5f, ad)) c -= 1;
        else if (ax >= __fmul_rn(whole - 7.5f, ad)) c += 1;
    }
    return (uint32_t)min(max(c, 0), 15);
}

// The scale of a block whose value of largest magnitude (the first one) is v.
EMB_DEV __half kv4_scale(float v) {
    const float d = fminf(fmaxf(v * -0.125f, -8160.0f), 8160.0f);
    uint32_t u = __float_as_uint(d);
    u = (u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u;      // 8 significant bits, ties to even
    return __float2half_rn(__uint_as_float(u));
}

// Eight elements of a block held by four neighbouring lanes: their codes as a word, and
// the block's scale. Called by whole warps.
EMB_DEV void kv4_block(float (&x)[8], uint32_t *word, __half *scale) {
    const int base = (threadIdx.x & 31) & ~3;
    // the largest and the smallest decide the scale unless they tie; z is NaN when some
    // element is no finite number
    float hi = x[0], lo = x[0], z = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        hi = fmaxf(hi, x[j]);
        lo = fminf(lo, x[j]);
        z = fmaf(x[j], 0.0f, z);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const float m = fmaxf(hi, -lo);
    __half d = kv4_scale(hi > -lo ? hi : lo);
    float df = __half2float(d), inv = __fdividef(1.0f, df);
    // ordinary blocks: |x / d| <= 8.04, so 1.5 * 2^23 + 8 + x / d has the code in its lower
    // bits, rounded to nearest; how far that was from x / d tells of borders
    uint32_t w = 0;
    float off = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float r = fmaf(x[j], inv, 12582920.0f);
        off = fmaxf(off, fabsf(fmaf(x[j], inv, 12582920.0f - r)));
        w += __float_as_uint(fminf(r, 12582927.0f)) << (4 * j);
    }
    w -= 0x4B400000u * 0x11111111u;
    // the others: no finite numbers, two largest of opposite signs, scales that saturate
    // or are no normal fp16 number, an element within 1e-5 of a border (x / d is 4e-6 off)
    const bool rare = z != z || hi == -lo || m > 65000.0f || m < 0.0005f || off > 0.49999f;
    if (__any_sync(0xffffffffu, rare)) {
        float am = 0.0f, first = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = x[j] != x[j] ? 0.0f : fminf(fmaxf(x[j], -3.402823466e38f), 3.402823466e38f);
            if (fabsf(x[j]) > am) { am = fabsf(x[j]); first = x[j]; }
        }
        float bm = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        // the first lane of the block that has it
        const unsigned mask = __ballot_sync(0xffffffffu, am == bm);
        d = kv4_scale(__shfl_sync(0xffffffffu, first, base + __ffs((mask >> base) & 0xfu) - 1));
        df = __half2float(d);
        inv = df != 0.0f ? __fdiv_rn(1.0f, df) : 0.0f;
        w = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) w |= (df != 0.0f ? kv4_code(x[j], df, inv) : 8u) << (4 * j);
    }
    *word = w;
    *scale = d;
}

// Store and read, one kernel per direction. Four lanes hold a block, each eight
// consecutive elements: one 32-bit key word, or one 16-bit piece of each of two value
// words; head_dim / 8 lanes hold a row of one head. A thread takes KV4_IO_ROWS rows
// in a row, so that their loads are under way together. Each row is read (written)
// once, 16 bytes a lane and load; bound by the conversions' integer instructions (issue
// slots 71 % used in the store, 80 % in the read): 14,000 fp16 rows of 8 heads of 128,
// 57 MB, 48 us into the cache and 20 us back. With two elements a lane and a division
// each it took 166 us for both.
// x: items (row, kv head, keys or values) of a row group; y: sequences.
constexpr int KV4_IO_THREADS = 256, KV4_IO_ROWS = 4;

template <typename T, int HD, bool STORE>
__global__ void __launch_bounds__(KV4_IO_THREADS) kv4_io_kernel(Kv4View c, Kv4Rows b, Kv4Io io, bool vec) {
    constexpr int LANES = HD / 8, NB = HD / 32, N = KV4_IO_ROWS;
    const Kv4Seq s = kv4_seq(b, blockIdx.y);
    const int lane = threadIdx.x % LANES, per_row = 2 * c.n_kv;
    const unsigned item = (blockIdx.x * KV4_IO_THREADS + threadIdx.x) / LANES;
    const int group_row = (int)(item / per_row), which = (int)(item - (unsigned)group_row * per_row);
    const bool is_v = which >= c.n_kv;           // neighbouring lanes: heads of the same tensor
    const int head = is_v ? which - c.n_kv : which;
    const int ps = 1 << c.page_shift, blk = lane >> 2, w4 = lane & 3;
    const int row0 = group_row * N, pos0 = s.len - s.rows + row0;
    const int64_t stride = is_v ? io.v_tok : io.k_tok;
    T *const mem0 = (T *)(is_v ? io.v : io.k) + (int64_t)(s.row0 + row0) * stride + head * (is_v ? io.v_head : io.k_head) +
                    lane * 8;
    uint8_t *const base = c.data + (size_t)head * c.chunk;
    const uint64_t page_bytes = (uint64_t)c.n_kv * c.chunk;
    const int32_t *table = b.table + (size_t)blockIdx.y * b.table_stride;
    uint8_t *group[N];               // the position's group of 16, or null
    T *mem[N];
    int in[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int pos = pos0 + i;
        const bool live = row0 + i < s.rows && pos >= 0 && pos < b.cap;
        const int page = live ? __ldg(table + (pos >> c.page_shift)) : -1;
        in[i] = pos & 15;
        group[i] = (unsigned)page < (unsigned)c.n_pages
                       ? base + (uint64_t)(uint32_t)page * page_bytes + ((pos & (ps - 1)) >> 4) * kv4_group(HD)
                       : nullptr;
        mem[i] = mem0 + i * stride;
    }
    if (!__any_sync(0xffffffffu, row0 < s.rows)) return;
    // where a position's codes and scale are: keys one word, values the halves of the
    // words g = 2 w4 and 2 w4 + 1
    auto codes = [&](int i) {
        return is_v ? group[i] + 8 * HD + (in[i] >> 1) * HD + (2 * w4) * (4 * NB) + 4 * blk + 2 * (in[i] & 1)
                    : group[i] + in[i] * (HD / 2) + w4 * (4 * NB) + 4 * blk;
    };
    auto scale = [&](int i) {
        return reinterpret_cast<__half *>(group[i] + 16 * HD) +
               (is_v ? 16 * NB + ((in[i] >> 1) * NB + blk) * 2 + (in[i] & 1) : in[i] * NB + blk);
    };
    float x[N][8];
    if (STORE) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (group[i]) load8(mem[i], vec, x[i]);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = j == 0 ? 1.0f : 0.0f;      // an ordinary block
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t w;
            __half d;
            kv4_block(x[i], &w, &d);
            if (!group[i]) continue;
            uint8_t *p = codes(i);
            if (is_v) {
                *reinterpret_cast<uint16_t *>(p) = (uint16_t)w;
                *reinterpret_cast<uint16_t *>(p + 4 * NB) = (uint16_t)(w >> 16);
            } else {
                *reinterpret_cast<uint32_t *>(p) = w;
            }
            if (w4 == 0) *scale(i) = d;
        }
    } else {
        uint32_t w[N];
        __half d[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            w[i] = 0;
            d[i] = __float2half_rn(0.0f);
            if (!group[i]) continue;
            const uint8_t *p = codes(i);
            w[i] = is_v ? *reinterpret_cast<const uint16_t *>(p) |
                              (uint32_t)*reinterpret_cast<const uint16_t *>(p + 4 * NB) << 16
                        : *reinterpret_cast<const uint32_t *>(p);
            d[i] = *scale(i);
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (!group[i]) continue;
            // (code - 8) * d, exact in fp16: dims 0,4 / 1,5 / 2,6 / 3,7
            const __half2 dd = __half2half2(d[i]);
            const uint32_t h0 = kp_low(w[i], dd), h1 = kp_high(w[i], dd), h2 = kp_low(w[i] >> 8, dd),
                           h3 = kp_high(w[i] >> 8, dd);
            const uint4 q = make_uint4(__byte_perm(h0, h1, 0x5410), __byte_perm(h2, h3, 0x5410),
                                       __byte_perm(h0, h1, 0x7632), __byte_perm(h2, h3, 0x7632));
            const __half2 *qh = reinterpret_cast<const __half2 *>(&q);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = __half22float2(qh[j]);
                x[i][2 * j] = f.x;
                x[i][2 * j + 1] = f.y;
            }
            if (sizeof(T) == 4) {
                float *o = reinterpret_cast<float *>(mem[i]);
                if (vec) {
                    reinterpret_cast<float4 *>(o)[0] = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
                    reinterpret_cast<float4 *>(o)[1] = make_float4(x[i][4], x[i][5], x[i][6], x[i][7]);
                } else
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = x[i][j];
            } else {
                __half *o = reinterpret_cast<__half *>(mem[i]);
                if (vec) {
                    *reinterpret_cast<uint4 *>(o) = q;
                } else
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = __float2half_rn(x[i][j]);
            }
        }
    }
}

template <typename T>
static int kv4_attention_launch(const Kv4AttnArgs &a, int hd, int *err, cudaStream_t st) {
    switch (kv4_kernel(sizeof(T), hd, a.b.n_tokens, a.max_q, a.group, a.c.n_kv, a.b.n_seqs)) {
    case KV4_FEW_4: return kv4_decode_hd<T, 1>(a, hd, st);
    case KV4_FEW_8: return kv4_decode_hd<T, 2>(a, hd, st);
    case KV4_MANY_1: return kv4_prompt_hd<T, 1>(a, hd, err, st);
    default: return kv4_prompt_hd<T, 2>(a, hd, err, st);
    }
}

// ------------------------------------------------------------ host checks ----

// the device that owns device memory p, or -1
static int kv4_device_of(const void *p) {
    cudaPointerAttributes attr;
    if (cudaPointerGetAttributes(&attr, p) != cudaSuccess) {
        cudaGetLastError();
        return -1;
    }
    return attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged ? attr.device : -1;
}

// the caller's device put back at the end of a call
struct DeviceScope {
    int prev = -1;
    bool ok = true;
    explicit DeviceScope(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) { cudaGetLastError(); prev = -1; }
        if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
        else prev = -1;
    }
    ~DeviceScope() { if (prev >= 0) cudaSetDevice(prev); }
};

static int kv4_shift(int page_size) {
    return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}
static bool kv4_shape_ok(int n_pages, int page_size, int n_kv, int hd) {
    return n_pages > 0 && kv4_shift(page_size) > 0 && (long long)n_pages * page_size <= 0x7FFFFFFFll && n_kv > 0 &&
           n_kv <= 1024 && (hd == 32 || hd == 64 || hd == 128);
}

// cache and batch into their device views; the device in *dev
static int kv4_views(const char *who, const EmberKv4Cache *cache, const EmberKv4Batch *batch, Kv4View *c, Kv4Rows *b,
                     int *dev) {
    if (!cache || !batch) return set_err("%s: null cache or batch", who);
    if (!kv4_shape_ok(cache->n_pages, cache->page_size, cache->n_kv_heads, cache->head_dim))
        return set_err("%s: cache of %d pages of %d positions, %d kv heads of %d is not supported (pages of 16, 32, 64 "
                       "or 128 positions, at most 2^31 - 1 in all; head_dim 32, 64 or 128)",
                       who, cache->n_pages, cache->page_size, cache->n_kv_heads, cache->head_dim);
    if (batch->n_seqs < 0 || batch->n_seqs > 65535) return set_err("%s: n_seqs %d is outside [0, 65535]", who, batch->n_seqs);
    if (batch->n_tokens < 0) return set_err("%s: negative n_tokens", who);
    if (batch->table_stride < 1) return set_err("%s: table_stride must be positive", who);
    if (batch->max_q < 0) return set_err("%s: negative max_q", who);
    if (!batch->q_start && batch->n_tokens != batch->n_seqs)
        return set_err("%s: without q_start every sequence has one row (%d rows, %d sequences)", who, batch->n_tokens,
                       batch->n_seqs);
    if ((uintptr_t)cache->data % 16) return set_err("%s: cache data is not 16-byte aligned", who);
    *dev = kv4_device_of(cache->data);
    if (*dev < 0) return set_err("%s: cache data is not device memory", who);
    if (batch->n_seqs > 0) {
        const void *p[3] = {batch->kv_len, batch->block_table, batch->q_start};
        for (int i = 0; i < 3; i++)
            if ((p[i] || i < 2) && (uintptr_t)p[i] % 4)
                return set_err("%s: the batch's arrays must be 4-byte aligned", who);
            else if ((p[i] || i < 2) && kv4_device_of(p[i]) != *dev)
                return set_err("%s: kv_len, block_table and q_start must be memory of the cache's device", who);
    }
    c->data = (uint8_t *)cache->data;
    c->n_pages = cache->n_pages;
    c->page_shift = kv4_shift(cache->page_size);
    c->n_kv = cache->n_kv_heads;
    c->chunk = kv4_chunk(cache->page_size, cache->head_dim);
    b->q_start = batch->q_start;
    b->kv_len = batch->kv_len;
    b->table = batch->block_table;
    b->n_seqs = batch->n_seqs;
    b->table_stride = batch->table_stride;
    b->n_tokens = batch->n_tokens;
    const long long cap = (long long)batch->table_stride * cache->page_size;
    b->cap = cap > 0x7FFF0000ll ? 0x7FFF0000 : (int)cap;      // tiles behind it stay within int
    return 0;
}

template <typename T, bool STORE>
static int kv4_io_launch(const Kv4View &c, const Kv4Rows &b, const Kv4Io &io, bool vec, int hd, int max_q,
                         cudaStream_t st) {
    const long long items = ((long long)max_q + KV4_IO_ROWS - 1) / KV4_IO_ROWS * 2 * c.n_kv * (hd / 8);
    const long long gx = (items + KV4_IO_THREADS - 1) / KV4_IO_THREADS;
    if (items > 0x7FFFFFFFll - KV4_IO_THREADS) return set_err("kv4: max_q %d is too large", max_q);
    const dim3 grid((unsigned)gx, (unsigned)b.n_seqs);
    switch (hd) {
    case 32: kv4_io_kernel<T, 32, STORE><<<grid, KV4_IO_THREADS, 0, st>>>(c, b, io, vec); break;
    case 64: kv4_io_kernel<T, 64, STORE><<<grid, KV4_IO_THREADS, 0, st>>>(c, b, io, vec); break;
    default: kv4_io_kernel<T, 128, STORE><<<grid, KV4_IO_THREADS, 0, st>>>(c, b, io, vec); break;
    }
    CK(cudaGetLastError());
    return 0;
}

template <bool STORE>
static int kv4_io(const char *who, const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Rows *rows,
                  cudaStream_t st) {
    Kv4View c;
    Kv4Rows b;
    int dev;
    if (kv4_views(who, cache, batch, &c, &b, &dev)) return 1;
    if (!rows) return set_err("%s: null rows", who);
    if (rows->dtype != EMBER_DT_F32 && rows->dtype != EMBER_DT_F16)
        return set_err("%s: dtype %d is not EMBER_DT_F32 or EMBER_DT_F16", who, rows->dtype);
    int max_q = batch->q_start ? batch->max_q : 1;
    if (max_q > b.n_tokens) max_q = b.n_tokens;
    if (b.n_seqs == 0 || max_q == 0) return 0;
    const size_t es = rows->dtype == EMBER_DT_F32 ? 4 : 2;
    if ((uintptr_t)rows->k % es || (uintptr_t)rows->v % es) return set_err("%s: k or v is not aligned to its type", who);
    if (kv4_device_of(rows->k) != dev || kv4_device_of(rows->v) != dev)
        return set_err("%s: k and v must be memory of the cache's device", who);
    if (rows->k_tok < 0 || rows->k_head < 0 || rows->v_tok < 0 || rows->v_head < 0)
        return set_err("%s: negative strides are not supported", who);
    // a lane's eight elements as 16-byte accesses
    const int64_t per = 16 / (int64_t)es;
    const bool vec = !((uintptr_t)rows->k % 16 || (uintptr_t)rows->v % 16 || rows->k_tok % per || rows->k_head % per ||
                       rows->v_tok % per || rows->v_head % per);
    Kv4Io io;
    io.k = const_cast<void *>(rows->k); io.v = const_cast<void *>(rows->v);
    io.k_tok = rows->k_tok; io.k_head = rows->k_head; io.v_tok = rows->v_tok; io.v_head = rows->v_head;
    DeviceScope scope(dev);
    if (!scope.ok) return set_err("%s: cannot select device %d", who, dev);
    if (rows->dtype == EMBER_DT_F32) return kv4_io_launch<float, STORE>(c, b, io, vec, cache->head_dim, max_q, st);
    return kv4_io_launch<__half, STORE>(c, b, io, vec, cache->head_dim, max_q, st);
}

}  // namespace emb

using namespace emb;

extern "C" size_t ember_cuda_kv4_bytes(int32_t n_pages, int32_t page_size, int32_t n_kv_heads, int32_t head_dim) {
    if (!kv4_shape_ok(n_pages, page_size, n_kv_heads, head_dim)) return 0;
    return (size_t)n_pages * n_kv_heads * kv4_chunk(page_size, head_dim);
}

extern "C" int ember_cuda_kv4_store(const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Rows *rows,
                                    void *stream) {
    return kv4_io<true>("kv4 store", cache, batch, rows, (cudaStream_t)stream);
}

extern "C" int ember_cuda_kv4_read(const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Rows *rows,
                                   void *stream) {
    return kv4_io<false>("kv4 read", cache, batch, rows, (cudaStream_t)stream);
}

extern "C" size_t ember_cuda_kv4_attention_workspace(const EmberKv4Cache *cache, int32_t n_heads, int32_t n_seqs,
                                                     int32_t max_q, int32_t max_kv) {
    if (!cache || n_heads < 1 || n_seqs < 1 || max_q < 1 || max_kv < 1 || cache->n_kv_heads < 1 ||
        n_heads % cache->n_kv_heads)
        return 0;
    return kv4_attention_workspace(cache->head_dim, max_kv);
}

int emb::kv4_attention(const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Attention *att, int *err,
                       cudaStream_t st) {
    const char *who = "kv4 attention";
    Kv4View c;
    Kv4Rows b;
    int dev;
    if (kv4_views(who, cache, batch, &c, &b, &dev)) return 1;
    if (!att) return set_err("%s: null arguments", who);
    if (att->dtype != EMBER_DT_F32 && att->dtype != EMBER_DT_F16)
        return set_err("%s: dtype %d is not EMBER_DT_F32 or EMBER_DT_F16", who, att->dtype);
    if (att->n_heads < 1 || att->n_heads % c.n_kv || att->n_heads > 65535)
        return set_err("%s: n_heads %d is not a multiple of n_kv_heads %d within 65535", who, att->n_heads, c.n_kv);
    if (!isfinite(att->scale)) return set_err("%s: scale must be finite", who);
    if (att->window < 0 || att->sinks < 0) return set_err("%s: window and sinks must not be negative", who);
    if (att->max_kv < 0) return set_err("%s: negative max_kv", who);
    int max_q = batch->q_start ? batch->max_q : 1;
    if (max_q > b.n_tokens) max_q = b.n_tokens;
    if (b.n_seqs == 0 || max_q == 0) return 0;
    const size_t es = att->dtype == EMBER_DT_F32 ? 4 : 2;
    if ((uintptr_t)att->q % es || (uintptr_t)att->out % es) return set_err("%s: q or out is not aligned to its type", who);
    if (kv4_device_of(att->q) != dev || kv4_device_of(att->out) != dev)
        return set_err("%s: q and out must be memory of the cache's device", who);
    if (att->q_tok < 0 || att->q_head < 0 || att->out_tok < 0 || att->out_head < 0)
        return set_err("%s: negative strides are not supported", who);
    const int hd = cache->head_dim;
    int max_kv = att->max_kv < b.cap ? att->max_kv : b.cap;
    const size_t need = kv4_attention_workspace(hd, max_kv);
    if (need) {
        if (att->workspace_bytes < need)
            return set_err("%s: workspace of %zu bytes, %zu needed", who, att->workspace_bytes, need);
        if ((uintptr_t)att->workspace % 16 || kv4_device_of(att->workspace) != dev)
            return set_err("%s: workspace must be 16-byte aligned memory of the cache's device", who);
    }
    DeviceScope scope(dev);
    if (!scope.ok) return set_err("%s: cannot select device %d", who, dev);
    Kv4AttnArgs a;
    a.c = c; a.b = b;
    a.q = att->q; a.out = att->out;
    a.q_tok = att->q_tok; a.q_head = att->q_head; a.out_tok = att->out_tok; a.out_head = att->out_head;
    a.n_heads = att->n_heads; a.group = att->n_heads / c.n_kv;
    a.scale = att->scale; a.max_kv = max_kv; a.max_q = max_q; a.window = att->window; a.sinks = att->sinks;
    a.ws = (float *)att->workspace;
    return att->dtype == EMBER_DT_F32 ? kv4_attention_launch<float>(a, hd, err, st)
                                      : kv4_attention_launch<__half>(a, hd, err, st);
}

extern "C" int ember_cuda_kv4_attention(const EmberKv4Cache *cache, const EmberKv4Batch *batch,
                                        const EmberKv4Attention *att, void *stream) {
    return kv4_attention(cache, batch, att, nullptr, (cudaStream_t)stream);
}

extern "C" int ember_cuda_kv4_status(const EmberKv4Cache *cache, void *stream) {
    const char *who = "kv4 status";
    if (!cache) return set_err("%s: null cache", who);
    const int dev = kv4_device_of(cache->data);
    if (dev < 0) return set_err("%s: cache data is not device memory", who);
    DeviceScope scope(dev);
    if (!scope.ok) return set_err("%s: cannot select device %d", who, dev);
    const cudaStream_t st = (cudaStream_t)stream;
    int code = 0;
    CK(cudaMemcpyFromSymbolAsync(&code, kv4_wait_error, sizeof(code), 0, cudaMemcpyDeviceToHost, st));
    CK(cudaStreamSynchronize(st));
    if (!code) return 0;
    const int none = 0;
    CK(cudaMemcpyToSymbolAsync(kv4_wait_error, &none, sizeof(none), 0, cudaMemcpyHostToDevice, st));
    CK(cudaStreamSynchronize(st));
    return set_err("kv4 attention: device wait timed out (code %d)", code);
}
