// kv4.cu — the paged 4-bit KV cache: store, read, and the host side of the
// attention over it (kernels in kv4_attn.cuh for few rows
// per sequence and kv4_prompt.cuh for many).
#include <cuda_runtime.h>

#include <math.h>

#include "kv4.cuh"
#include "kv4_prompt.cuh"
#include "runtime_internal.cuh"

namespace emb {

struct Kv4Io {
    void *k, *v;
    int64_t k_tok, k_head, v_tok, v_head;
};

EMB_DEV void load4(const float *p, bool vec, float (&x)[4]) {
    if (vec) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = p[j];
    }
}
EMB_DEV void load4(const __half *p, bool vec, float (&x)[4]) {
    if (vec) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = __half2float(p[j]);
    }
}

// code of x for scale d: floor(x / d + 8.5) in exact arithmetic. The division and
// the addition round, so the result can be one off where x / d lies next to a
// border (c - 8.5); a border times d has 13 significant bits, exact in fp32, so
// comparing x with the borders around the first guess settles it.
EMB_DEV uint32_t kv4_code(float x, float d) {
    const float ax = d < 0.0f ? -x : x, ad = fabsf(d);
    float c = floorf(__fadd_rn(__fdiv_rn(ax, ad), 8.5f));
    c = fminf(fmaxf(c, 0.0f), 15.0f);
    if (ax < __fmul_rn(c - 8.5f, ad)) c -= 1.0f;
    else if (ax >= __fmul_rn(c - 7.5f, ad)) c += 1.0f;
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);
}

// The scale of a block whose value of largest magnitude (the first one) is v.
EMB_DEV __half kv4_scale(float v) {
    const float d = fminf(fmaxf(v * -0.125f, -8160.0f), 8160.0f);
    uint32_t u = __float_as_uint(d);
    u = (u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u;      // 8 significant bits, ties to even
    return __float2half_rn(__uint_as_float(u));
}

// Store and read, one kernel per direction. Eight lanes hold a block, each four
// consecutive elements and so one 16-bit piece of a key word or of a value row;
// head_dim / 4 lanes hold a row of one head. Bound by memory: each row is read
// (written) once, 16 bytes a lane for fp32 rows.
// x: items (row, kv head, keys or values); y: sequences.
constexpr int KV4_IO_THREADS = 256;

template <typename T, int HD, bool STORE>
__global__ void __launch_bounds__(KV4_IO_THREADS) kv4_io_kernel(Kv4View c, Kv4Rows b, Kv4Io io, bool vec) {
    constexpr int LANES = HD / 4, NB = HD / 32;
    const Kv4Seq s = kv4_seq(b, blockIdx.y);
    const int lane = threadIdx.x % LANES;
    const long long item = ((long long)blockIdx.x * KV4_IO_THREADS + threadIdx.x) / LANES;
    const int per_row = 2 * c.n_kv;
    const long long row = item / per_row;
    // no lane leaves before the shuffles: lanes of other items share the warp
    bool live = row < s.rows;
    const int which = (int)(item % per_row), head = which >> 1;
    const bool is_v = which & 1;
    const long long pos = (long long)s.len - s.rows + row;
    live = live && pos >= 0 && pos < b.cap;
    const int page = live ? kv4_page(c, b, blockIdx.y, (int)pos) : -1;
    live = page >= 0;
    const int slot = (int)(pos & ((1 << c.page_shift) - 1)), in = slot & 15;
    uint8_t *chunk = live ? kv4_chunk_ptr(c, page, head) : nullptr;
    const int blk = lane >> 3, g = lane & 7;
    uint16_t *code = nullptr;
    __half *scale = nullptr;
    if (live) {
        uint8_t *group = chunk + (slot >> 4) * kv4_group(HD);
        const int pair = in >> 1, odd = in & 1;
        code = reinterpret_cast<uint16_t *>(
            group + (is_v ? 8 * HD + pair * HD + g * (4 * NB) + 4 * blk + 2 * odd
                          : in * (HD / 2) + (g >> 1) * (4 * NB) + 4 * blk + 2 * (g & 1)));
        scale = reinterpret_cast<__half *>(group + 16 * HD) + (is_v ? 16 * NB + (pair * NB + blk) * 2 + odd : in * NB + blk);
    }
    const long long tok = s.row0 + row;
    T *mem = nullptr;
    if (live)
        mem = is_v ? (T *)io.v + tok * io.v_tok + head * io.v_head + lane * 4
                   : (T *)io.k + tok * io.k_tok + head * io.k_head + lane * 4;
    if (STORE) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (live) load4(mem, vec, x);
        float m = 0.0f, first = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = x[j] != x[j] ? 0.0f : fminf(fmaxf(x[j], -3.402823466e38f), 3.402823466e38f);
            if (fabsf(x[j]) > m) { m = fabsf(x[j]); first = x[j]; }
        }
        float bm = m;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
        const unsigned mask = __ballot_sync(0xffffffffu, m == bm);
        const int base = (threadIdx.x & 31) & ~7;
        const int src = base + __ffs((mask >> base) & 0xffu) - 1;
        const __half d = kv4_scale(__shfl_sync(0xffffffffu, first, src));
        const float df = __half2float(d);
        if (!live) return;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w |= (df != 0.0f ? kv4_code(x[j], df) : 8u) << (4 * j);
        *code = (uint16_t)w;
        if (g == 0) *scale = d;
    } else {
        if (!live) return;
        const uint32_t w = *code;
        const float d = __half2float(*scale);
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (float)((int)((w >> (4 * j)) & 15u) - 8) * d;
        if (sizeof(T) == 4) {
            float *o = reinterpret_cast<float *>(mem);
            if (vec) *reinterpret_cast<float4 *>(o) = make_float4(x[0], x[1], x[2], x[3]);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = x[j];
        } else {
            __half *o = reinterpret_cast<__half *>(mem);
            __half2 h[2] = {__floats2half2_rn(x[0], x[1]), __floats2half2_rn(x[2], x[3])};   // exact
            if (vec) *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<uint2 *>(h);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = __float2half_rn(x[j]);
        }
    }
}

// Up to this many rows (tokens x query heads of a kv head) a sequence's rows are taken
// eight at a time, the cache read once for each eight; beyond, 128 at a time.
constexpr int KV4_FEW_ROWS = 16;

template <typename T>
static int kv4_attention_launch(const Kv4AttnArgs &a, int hd, cudaStream_t st) {
    const long long rows = (long long)a.max_q * a.group;
    if (rows > KV4_FEW_ROWS) return kv4_prompt_hd<T>(a, hd, st);
    return rows <= 4 ? kv4_decode_hd<T, 1>(a, hd, st) : kv4_decode_hd<T, 2>(a, hd, st);
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
    b->cap = cap > 0x7FFFFFFFll ? 0x7FFFFFFF : (int)cap;
    return 0;
}

template <typename T, bool STORE>
static int kv4_io_launch(const Kv4View &c, const Kv4Rows &b, const Kv4Io &io, bool vec, int hd, int max_q,
                         cudaStream_t st) {
    const long long items = (long long)max_q * 2 * c.n_kv * (hd / 4);
    const long long gx = (items + KV4_IO_THREADS - 1) / KV4_IO_THREADS;
    if (gx > 0x7FFFFFFFll) return set_err("kv4: max_q %d is too large", max_q);
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
    const size_t w = 4 * es;      // a lane's four elements as one access
    const bool vec = !((uintptr_t)rows->k % w || (uintptr_t)rows->v % w || rows->k_tok % 4 || rows->k_head % 4 ||
                       rows->v_tok % 4 || rows->v_head % 4);
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

extern "C" int ember_cuda_kv4_attention(const EmberKv4Cache *cache, const EmberKv4Batch *batch,
                                        const EmberKv4Attention *att, void *stream) {
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
    return att->dtype == EMBER_DT_F32 ? kv4_attention_launch<float>(a, hd, (cudaStream_t)stream)
                                      : kv4_attention_launch<__half>(a, hd, (cudaStream_t)stream);
}
