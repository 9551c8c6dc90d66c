// sample_rows.cu — one draw per row of a batch of logits.
//
// The tokens of a row are ordered by (logit descending, index ascending); each
// has the weight w = exp((logit - max) / temperature), rounded to a multiple of
// 2^-44 and held as an integer. Every truncation keeps a prefix of that order, so
// the kept weight is the smallest of the prefixes' weights, and the draw is again
// a prefix: the first token whose running weight reaches floor(u * kept) + 1. All
// of them ask one question -- where does a running sum (of weights or of ones)
// reach a target -- answered by a radix descent over the 64-bit keys
// (descending logit bits, index), eight bits a pass. The sums are integers:
// no order of additions can change a token.
#include <cuda_runtime.h>

#include "common.cuh"
#include "ember_kv4.h"
#include "runtime_internal.cuh"

namespace emb {

constexpr int SR_THREADS = 1024;

EMB_DEV float sr_logit(float v) { return v != v ? -INFINITY : v; }
// ascending keys are descending logits (-0 and +0 alike)
EMB_DEV uint32_t sr_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u >> 31) ? u : ~(u | 0x80000000u);
}
EMB_DEV double sr_weight(float l, float mx, double t) {
    if (l == mx) return 1.0;
    if (l == -INFINITY) return 0.0;
    return exp(((double)l - (double)mx) / t);
}
EMB_DEV unsigned long long sr_units(double w) { return (unsigned long long)__double2ll_rn(w * 17592186044416.0); }

template <typename T>
__global__ void __launch_bounds__(SR_THREADS) sample_rows_kernel(EmberSampleRows a) {
    __shared__ unsigned long long hist[256], s_sum[32], s_out[4];
    __shared__ float s_v[32];
    __shared__ int s_i[32];
    const int tid = threadIdx.x, row = blockIdx.x, n = a.vocab;
    const T *x = (const T *)a.logits + (int64_t)row * a.stride;
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    float mx = -INFINITY;
    int mi = 0x7FFFFFFF;
    for (int i = tid; i < n; i += SR_THREADS) {
        const float v = sr_logit(widen(x[i]));
        if (v > mx) { mx = v; mi = i; }
    }
    auto take = [&](float v, int i) {
        if (v > mx || (v == mx && i < mi)) { mx = v; mi = i; }
    };
    for (int o = 16; o; o >>= 1) take(__shfl_xor_sync(~0u, mx, o), __shfl_xor_sync(~0u, mi, o));
    if (tid % 32 == 0) { s_v[tid / 32] = mx; s_i[tid / 32] = mi; }
    __syncthreads();
    mx = s_v[tid % 32];
    mi = s_i[tid % 32];
    for (int o = 16; o; o >>= 1) take(__shfl_xor_sync(~0u, mx, o), __shfl_xor_sync(~0u, mi, o));
    if (!(temp > 0.0f) || mx == -INFINITY) {
        if (tid == 0) a.out[row] = mx == -INFINITY ? 0 : mi;
        return;
    }
    const double t = (double)temp;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    // whole weight and the weight of what min_p keeps
    auto block_sum = [&](unsigned long long v) {
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        __syncthreads();
        if (tid % 32 == 0) s_sum[tid / 32] = v;
        __syncthreads();
        v = s_sum[tid % 32];
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    };
    const bool use_min = min_p > 0.0f && min_p < 1.0f;
    unsigned long long total = 0, kept = 0;
    for (int i = tid; i < n; i += SR_THREADS) {
        const double w = sr_weight(sr_logit(widen(x[i])), mx, t);
        total += sr_units(w);
        if (!use_min || w >= (double)min_p) kept += sr_units(w);
    }
    total = block_sum(total);
    kept = block_sum(kept);
    // the first token (in order) at which the running sum reaches target: its
    // index, and the running weight there
    auto find = [&](unsigned long long target, bool count, unsigned long long *weight) {
        unsigned long long prefix = 0, acc = 0, wacc = 0;
        for (int shift = 56; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            unsigned long long below = 0;     // weight before the prefix's range
            for (int i = tid; i < n; i += SR_THREADS) {
                const float l = sr_logit(widen(x[i]));
                const unsigned long long key = ((unsigned long long)sr_key(l) << 32) | (unsigned)i;
                if (shift == 56 || (key >> (shift + 8)) == prefix)
                    atomicAdd(&hist[(key >> shift) & 255], count ? 1ull : sr_units(sr_weight(l, mx, t)));
            }
            __syncthreads();
            if (tid == 0) {
                int b = 0;
                for (; b < 255 && acc + hist[b] < target; b++) acc += hist[b];
                s_out[0] = (prefix << 8) | b;
                s_out[1] = acc;
            }
            __syncthreads();
            prefix = s_out[0];
            acc = s_out[1];
            (void)below;
        }
        for (int i = tid; i < n; i += SR_THREADS) {
            const float l = sr_logit(widen(x[i]));
            const unsigned long long key = ((unsigned long long)sr_key(l) << 32) | (unsigned)i;
            if (key <= prefix) wacc += sr_units(sr_weight(l, mx, t));
        }
        *weight = block_sum(wacc);
        return (int)(prefix & 0xFFFFFFFFu);
    };
    unsigned long long w;
    if (k > 0 && k < n) {
        find((unsigned long long)k, true, &w);
        kept = min(kept, w);
    }
    if (top_p > 0.0f && top_p < 1.0f) {
        const unsigned long long target = (unsigned long long)ceil((double)top_p * (double)total);
        find(max(1ull, min(target, total)), false, &w);
        kept = min(kept, w);
    }
    const float u = a.u[row];
    const double r = (u > 0.0f ? (double)fminf(u, 1.0f) : 0.0) * (double)kept;
    const unsigned long long before = min((unsigned long long)r, kept - 1);
    const int tok = find(before + 1, false, &w);
    if (tid == 0) a.out[row] = tok;
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
    if (a.dtype == EMBER_DT_F32) sample_rows_kernel<float><<<a.n_rows, SR_THREADS, 0, st>>>(a);
    else sample_rows_kernel<__half><<<a.n_rows, SR_THREADS, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (prev != dev) cudaSetDevice(prev);
    if (e != cudaSuccess) return set_err("%s: %s", who, cudaGetErrorString(e));
    return 0;
}
