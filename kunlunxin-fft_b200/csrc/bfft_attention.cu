// bfft_attention.cu -- attention of ragged query rows over a paged 8-bit cache.
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(t q_i . k_j - m_i),
// over the tokens j that row i sees, with the running maximum m_i and sum kept
// in 32 bits while the tokens pass once.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/bfft.h"
#include "bfft_cache.cuh"
#include "bfft_kernels.cuh"

using namespace bfft;

namespace bfft {

struct AttentionArgs {
    CacheView cache;
    SequenceView seq;  // lens: tokens of each sequence in the cache
    const void* q;
    void* out;
    float* lse;
    int64_t qt, qh, ot, oh;
    int q_heads, group;  // group = q_heads / kv_heads
    int causal, window;
    float scale_log2;    // softmax_scale * log2(e)
};

// A warp per (row, query head), a token at a time, lanes over the dimensions.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) k_attention_rows(AttentionArgs a) {
    const int lane = threadIdx.x & 31, dim = a.cache.dim;
    const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t row = i / a.q_heads;
    if (row >= a.seq.tokens) return;
    const int head = (int)(i - row * a.q_heads), kv = head / a.group;
    const int s = find_sequence(a.seq.starts, a.seq.seqs, row);
    const int64_t t0 = a.seq.starts[s], t1 = a.seq.starts[s + 1], len = a.seq.lens[s];
    const int64_t pos = len - (t1 - row);
    int64_t hi = a.causal ? pos + 1 : len, lo = 0;
    if (a.window > 0 && pos - a.window + 1 > lo) lo = pos - a.window + 1;
    if (row < t0 || row >= t1) hi = 0;
    float q[8], o[8];
    const T* x = static_cast<const T*>(a.q) + row * a.qt + head * a.qh;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        q[d] = d * 32 + lane < dim ? to_f32(x[d * 32 + lane]) : 0.f;
        o[d] = 0.f;
    }
    float m = -INFINITY, sum = 0.f;
    for (int64_t j = lo; j < hi; ++j) {
        const int64_t page = page_of(a.seq, a.cache, s, j);
        if (page < 0) continue;
        const int64_t block = page * a.cache.kv_heads + kv;
        const int64_t at = ((block << a.cache.page_log2) + (j & (((int64_t)1 << a.cache.page_log2) - 1))) * dim;
        float dot = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d)
            if (d * 32 + lane < dim) dot += q[d] * code_value<CODE>(a.cache.k[at + d * 32 + lane]);
#pragma unroll
        for (int w = 16; w; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
        const float z = dot * a.cache.k_scale[block] * a.scale_log2;
        const float top = fmaxf(m, z), down = exp2f(m - top), p = exp2f(z - top), pv = p * a.cache.v_scale[block];
        m = top;
        sum = sum * down + p;
#pragma unroll
        for (int d = 0; d < 8; ++d)
            if (d * 32 + lane < dim) o[d] = o[d] * down + pv * code_value<CODE>(a.cache.v[at + d * 32 + lane]);
    }
    T* y = static_cast<T*>(a.out) + row * a.ot + head * a.oh;
    const bool none = sum == 0.f;  // no token seen (a NaN sum is not none)
#pragma unroll
    for (int d = 0; d < 8; ++d)
        if (d * 32 + lane < dim) y[d * 32 + lane] = from_f32<T>(none ? 0.f : o[d] / sum);
    if (a.lse && lane == 0) a.lse[row * a.q_heads + head] = none ? -INFINITY : (m + log2f(sum)) * 0.69314718f;
}

}  // namespace bfft

namespace {

bfft_status fail(bfft_status st, const char* fmt, ...) {
    char buf[384];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);  // reported by bfft_last_error()
    return st;
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

bfft_status check(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, const bfft_attention_desc* d) {
    if (!cache || !seqs || !d || !d->q || !d->out) return fail(BFFT_ERR_VALUE, "null pointer");
    bfft_status st = check_cache(cache);
    if (st == BFFT_OK) st = check_sequences(seqs);
    if (st != BFFT_OK) return st;
    if (d->type != BFFT_F16 && d->type != BFFT_BF16)
        return fail(BFFT_ERR_UNSUPPORTED, "queries must be float16 or bfloat16, got type %lld", (long long)d->type);
    if (d->q_heads < 1 || d->q_heads % cache->kv_heads || d->q_heads > 0xffffff)
        return fail(BFFT_ERR_SHAPE, "%lld query heads are no multiple of %lld kv heads", (long long)d->q_heads,
                    (long long)cache->kv_heads);
    if (d->window < 0 || d->window > 0x7fffffffLL) return fail(BFFT_ERR_VALUE, "bad window %lld", (long long)d->window);
    if (!std::isfinite(d->softmax_scale)) return fail(BFFT_ERR_VALUE, "softmax_scale must be finite");
    if (!aligned(d->q, 2) || !aligned(d->out, 2) || !aligned(d->lse, 4)) return fail(BFFT_ERR_VALUE, "misaligned pointer");
    return BFFT_OK;
}

struct Device {
    int prev = -1;
    bool ok = true, changed = false;
    explicit Device(int64_t dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) ok = cudaSetDevice((int)dev) == cudaSuccess;
        changed = ok && prev != dev;
    }
    ~Device() {
        if (changed && prev >= 0) cudaSetDevice(prev);
    }
};

template <typename T>
void rows_code(int64_t code, const AttentionArgs& a, unsigned grid, cudaStream_t s) {
    if (code == BFFT_CODE_INT8)
        k_attention_rows<T, kCodeInt8><<<grid, 256, 0, s>>>(a);
    else
        k_attention_rows<T, kCodeE4m3><<<grid, 256, 0, s>>>(a);
}

}  // namespace

extern "C" bfft_status bfft_cache_attention_workspace(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                                      const bfft_attention_desc* d, size_t* bytes) {
    if (!bytes) return fail(BFFT_ERR_VALUE, "null pointer");
    const bfft_status st = check(cache, seqs, d);
    if (st != BFFT_OK) return st;
    *bytes = 0;
    return BFFT_OK;
}

extern "C" bfft_status bfft_cache_attention(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                            const bfft_attention_desc* d, void* stream) {
    const bfft_status st = check(cache, seqs, d);
    if (st != BFFT_OK) return st;
    if (seqs->tokens == 0) return BFFT_OK;
    AttentionArgs a;
    a.cache = cache_view(cache);
    a.seq = sequence_view(seqs);
    a.q = d->q;
    a.out = d->out;
    a.lse = static_cast<float*>(d->lse);
    a.qt = d->q_token, a.qh = d->q_head, a.ot = d->o_token, a.oh = d->o_head;
    a.q_heads = (int)d->q_heads;
    a.group = (int)(d->q_heads / cache->kv_heads);
    a.causal = d->causal != 0;
    a.window = (int)d->window;
    a.scale_log2 = (float)(d->softmax_scale * 1.4426950408889634);
    const int64_t blocks = (seqs->tokens * d->q_heads + 7) / 8;
    if (blocks > 0x7fffffffLL) return fail(BFFT_ERR_SHAPE, "too many rows: %lld", (long long)seqs->tokens);
    Device g(d->device);
    if (!g.ok) return fail(BFFT_ERR_CUDA, "cannot select device %lld", (long long)d->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    count_launches(1);
    if (d->type == BFFT_F16)
        rows_code<__half>(cache->code, a, (unsigned)blocks, s);
    else
        rows_code<__nv_bfloat16>(cache->code, a, (unsigned)blocks, s);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BFFT_OK : fail(BFFT_ERR_CUDA, "cache_attention: %s", cudaGetErrorString(e));
}
