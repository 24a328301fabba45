// bfft_attention.cu -- attention of ragged query rows over a paged 8-bit cache.
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(t q_i . k_j - m_i),
// over the tokens j that row i sees, with the running maximum m_i and sum kept
// in 32 bits while the tokens pass once.
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>

#include "../../include/bfft.h"
#include "bfft_async.cuh"
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
    int q_packs, o_packs;  // rows of q / out start on 16 bytes
};

}  // namespace bfft

#include "bfft_attention_split.cuh"
#include "bfft_attention_tiles.cuh"

namespace {

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

using EncodeTiledFn = PFN_cuTensorMapEncodeTiled_v12000;

EncodeTiledFn encoder() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// The codes as [pages][kv_heads * page * dim / 128][128 bytes], boxes of 16 tokens,
// 128-byte swizzle (heads of 64, 128 or 256 elements: whole lines).
bool encode_codes(CUtensorMap* m, const void* codes, const bfft_cache_desc* c) {
    EncodeTiledFn enc = encoder();
    if (!enc) return false;
    const cuuint64_t lines = (cuuint64_t)(c->kv_heads * c->page * c->dim / 128);
    cuuint64_t dims[3] = {128, lines, (cuuint64_t)c->pages};
    cuuint64_t strides[2] = {128, 128 * lines};
    cuuint32_t box[3] = {128, (cuuint32_t)(c->dim / 8), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count(int64_t device) {
    static std::atomic<int> counts[64];
    if (device < 0 || device >= 64) return 148;
    const int dev = (int)device;
    int n = counts[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 148;
        }
        counts[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Tokens that a row tile of `tile` query tokens sees at most.
int64_t seen_cover(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int tile,
                   int align) {
    int64_t cover = q->max_pages * c->page;
    if (d->causal && d->window > 0) {
        const int64_t w = d->window + tile - 1 + align - 1;
        if (w < cover) cover = w;
    }
    return cover;
}

// Chunks and slots of the kernel for many rows.
struct TilePlan {
    int tile_tokens, by_token, chunk, chunks;
    int64_t slots, ctas;
    size_t bytes;
};

// How a call is cut: row tiles and chunks of the token axis.
struct SplitPlan {
    int nt, tile_tokens, token_tiles, by_token, chunk, chunks, cluster, entries;
    int64_t slots, ctas;
    size_t bytes;
};

SplitPlan plan_split(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int sms) {
    SplitPlan p;
    const int64_t group = d->q_heads / c->kv_heads;
    const int64_t each = q->tokens / q->seqs + (q->tokens % q->seqs != 0);  // rows of a sequence, about
    p.nt = each * group > 8 && c->dim <= 128 ? 2 : 1;
    const int64_t rows = 8 * p.nt;
    p.tile_tokens = group <= rows ? (int)(rows / group) : 1;
    p.token_tiles = group <= rows ? 1 : (int)((group + rows - 1) / rows);
    const int64_t runs = q->tokens / p.tile_tokens + q->seqs;
    p.by_token = q->tokens <= runs;
    p.slots = p.by_token ? q->tokens : runs;
    const int64_t cover = seen_cover(c, q, d, p.tile_tokens, 16);
    const int64_t tiles = (q->tokens + p.tile_tokens - 1) / p.tile_tokens;
    const int64_t units = tiles * p.token_tiles * c->kv_heads, resident = 3 * (int64_t)sms;
    // Where rows are many, chunks of 2048 tokens (512..4096 measure alike for 64 ragged
    // sequences).  Where they are few the table's width is shared out over a number of
    // CTAs that is counted as if three were resident on an SM (two are with 16 rows a
    // tile, one with heads over 128) and as if row tiles were full (those of sequences of
    // few rows are not: a tile's rows are one sequence's): "waves" times that many.  One
    // sequence of 131001 tokens, whose tiles are full: 71.6 us with 1, 75.8 with 2, 84.0
    // with 3, so 1, as a further wave's start costs more than it hides; 16 of 2000..8000
    // tokens, whose 4-row tiles are half full: 63.5, 59.4 and 69.6, so 2 for many
    // sequences.  The table's width is all that the host knows of the lengths: with a
    // table of 131072 tokens one row over 700 takes 21.5 us (14.3 with a table of 700,
    // timed with a cold L2), 8 over 4000 74.8 (37.9).
    const int64_t waves = q->seqs > 8 ? 2 : 1;
    int64_t chunks = units >= 2 * resident ? (cover + 2047) / 2048 : waves * resident / units;
    if (chunks < 1) chunks = 1;
    int64_t chunk = (cover + chunks - 1) / chunks;
    chunk = (chunk + 31) / 32 * 32;
    if (chunk < 256) chunk = 256;
    if (chunk > 4096) chunk = 4096;
    // Few rows over a short axis: eight chunks at most, one cluster that joins them
    // itself (8 row tiles over 704 tokens 10.1 us a call, by two launches 14.7; over 2000
    // tokens 12.3 by either, over 4000 15.4 and 12.7; 64 row tiles 28.7 and 22.6: a
    // cluster's CTAs keep their places until the last is done)
    const bool brief = units <= 32 && cover <= 2048;
    if (brief) {
        chunk = (cover + 7) / 8;
        chunk = (chunk + 31) / 32 * 32;
        if (chunk < 128) chunk = 128;
    }
    // The parts of many rows over a wide table (the plan knows the table's width, not the
    // lengths) are kept to 256 MB by longer chunks, as far as shared memory holds their
    // pages' scales (4.4 GB without: 512 sequences of 4 rows of 64 heads, 131072 tokens wide)
    const int64_t part = q->tokens * d->q_heads * (c->dim + 2) * 4, budget = (int64_t)256 << 20;
    if (!brief && (cover + chunk - 1) / chunk * part > budget) {
        const int64_t n = part < budget ? budget / part : 1;
        const int64_t room = (kSplitSmemMost - split_smem((int)c->dim, 8 * p.nt, 0)) / (int64_t)(sizeof(BlockScale) + 4);
        int64_t most = (room - 2) * c->page;
        if (most > 1 << 20) most = 1 << 20;
        chunk = ((cover + n - 1) / n + 31) / 32 * 32;
        if (chunk > most) chunk = most / 32 * 32;
    }
    p.entries = (int)(chunk / c->page + 2);
    p.chunk = (int)chunk;
    const int64_t n = (cover + chunk - 1) / chunk;
    p.chunks = (int)n;
    p.cluster = brief && n > 1;
    p.ctas = p.slots * p.token_tiles * c->kv_heads * n;
    p.bytes = n > 1 && !p.cluster ? (size_t)(q->tokens * d->q_heads * n) * (size_t)(c->dim + 2) * 4 : 0;
    return p;
}

// Whether a call is one for the tensor-core tiles: with 48 rows or more to a kv
// head (16 rows of 32 heads over 16384 tokens: 44 us, split kernel 73; 8 rows: 58
// by either) and enough work to pay for a CTA's start and its 128-row halves, some
// 3 million (query head, token) pairs of 128 dimensions: 40 rows of 32 heads over
// 900 tokens 30 us by the split kernel and 42 by this, 128 rows 58 and 48.  The rows
// are the mean of the call's sequences, so one kernel takes a prompt and single tokens
// together: a prompt of 4096 rows with 255 single tokens of 4096, 32 heads, 1139 us
// (apart 234 and 392), of 512 rows 661 (33 and 392).  Heads over 128 (S and O of two
// halves are more than tensor memory) and groups over 128 stay with the split kernel:
// 2 x 2048 rows of 16 heads of 256 over 8192 and 16384 tokens 10.6 ms, of 128 0.45.
bool use_tiles(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d) {
    const int64_t group = d->q_heads / c->kv_heads, each = q->tokens / q->seqs;
    if (c->dim > 128 || group > 128 || each * group < 48) return false;
    const double pairs = (double)q->tokens * (double)d->q_heads * (double)seen_cover(c, q, d, 1, 1);
    return pairs * (double)c->dim >= 3.0e6 * 128;
}

TilePlan plan_tiles(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int sms) {
    TilePlan p;
    const int64_t group = d->q_heads / c->kv_heads;
    p.tile_tokens = (int)(256 / group);
    const int64_t runs = q->tokens / p.tile_tokens + q->seqs;
    p.by_token = q->tokens <= runs;
    p.slots = p.by_token ? q->tokens : runs;
    const int64_t cover = seen_cover(c, q, d, p.tile_tokens, 128);
    const int64_t units = (q->tokens + p.tile_tokens - 1) / p.tile_tokens * c->kv_heads;
    int64_t chunks = units >= sms ? 1 : sms / units;
    int64_t chunk = (cover + chunks - 1) / chunks;
    if (chunk < 512) chunk = 512;
    chunk = (chunk + 127) / 128 * 128;
    if (chunk > 0x7fffff80LL) chunk = 0x7fffff80LL;
    p.chunk = (int)chunk;
    p.chunks = (int)((cover + chunk - 1) / chunk);
    p.ctas = p.slots * c->kv_heads * p.chunks;
    p.bytes = p.chunks > 1 ? (size_t)(q->tokens * d->q_heads * p.chunks) * (size_t)(c->dim + 2) * 4 : 0;
    return p;
}

template <int DP, typename T, int CODE>
cudaError_t launch_tiles(const TileArgs& a, const TilePlan& p, cudaStream_t s) {
    static std::atomic<bool> ready[64];
    using G = TileGeo<DP>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    auto* kernel = k_attention_tiles<DP, T, CODE>;
    if (!ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e != cudaSuccess) return e;
        ready[dev].store(true, std::memory_order_release);
    }
    return launch_dependent(kernel, (unsigned)p.ctas, G::THREADS, G::SMEM, s, a);
}

template <typename T>
cudaError_t run_join(const SplitArgs& a, cudaStream_t s) {
    const unsigned rows = (unsigned)(a.a.seq.tokens * a.a.q_heads);
    return a.chunks > 16 ? launch_dependent(k_attention_join<T, 16>, rows, 512, 0, s, a)
                         : launch_dependent(k_attention_join<T, 4>, rows, 128, 0, s, a);
}

template <typename T>
cudaError_t run_tiles(const TileArgs& a, const TilePlan& p, const bfft_cache_desc* c, cudaStream_t s) {
    cudaError_t e;
    if (c->dim <= 64)
        e = c->code == BFFT_CODE_INT8 ? launch_tiles<64, T, kCodeInt8>(a, p, s) : launch_tiles<64, T, kCodeE4m3>(a, p, s);
    else
        e = c->code == BFFT_CODE_INT8 ? launch_tiles<128, T, kCodeInt8>(a, p, s)
                                      : launch_tiles<128, T, kCodeE4m3>(a, p, s);
    if (e != cudaSuccess || p.chunks == 1) return e;
    SplitArgs j{};
    j.a = a.a;
    j.parts = a.parts;
    j.stats = a.stats;
    j.chunks = a.chunks;
    return run_join<T>(j, s);
}

template <int DP, bool EXACT, int NT, typename T, int CODE>
cudaError_t launch_split(const SplitArgs& a, const SplitPlan& p, const CUtensorMap& km, const CUtensorMap& vm,
                         cudaStream_t s) {
    static std::atomic<bool> ready[64];
    using G = SplitGeo<DP, EXACT, NT>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    auto* kernel = k_attention_split<DP, EXACT, NT, T, CODE>;
    if (!ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmemMost);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     (int)cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        ready[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3((unsigned)p.ctas);
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = split_smem(a.a.cache.dim, G::ROWS, a.entries);
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_dependent
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.chunks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, km, vm);
}

template <typename T, int CODE>
cudaError_t split_shape(const SplitArgs& a, const SplitPlan& p, const CUtensorMap& km, const CUtensorMap& vm,
                        cudaStream_t s) {
    const int dim = a.a.cache.dim;
    if (dim == 64)
        return p.nt == 1 ? launch_split<64, true, 1, T, CODE>(a, p, km, vm, s)
                         : launch_split<64, true, 2, T, CODE>(a, p, km, vm, s);
    if (dim == 128)
        return p.nt == 1 ? launch_split<128, true, 1, T, CODE>(a, p, km, vm, s)
                         : launch_split<128, true, 2, T, CODE>(a, p, km, vm, s);
    if (dim == 256) return launch_split<256, true, 1, T, CODE>(a, p, km, vm, s);
    if (dim < 128)
        return p.nt == 1 ? launch_split<128, false, 1, T, CODE>(a, p, km, vm, s)
                         : launch_split<128, false, 2, T, CODE>(a, p, km, vm, s);
    return launch_split<256, false, 1, T, CODE>(a, p, km, vm, s);
}

template <typename T>
cudaError_t run_split(const SplitArgs& a, const SplitPlan& p, const bfft_cache_desc* c, cudaStream_t s) {
    CUtensorMap km{}, vm{};
    if (c->dim == 64 || c->dim == 128 || c->dim == 256)
        if (!encode_codes(&km, c->k, c) || !encode_codes(&vm, c->v, c)) return cudaErrorNotSupported;
    cudaError_t e = c->code == BFFT_CODE_INT8 ? split_shape<T, kCodeInt8>(a, p, km, vm, s)
                                              : split_shape<T, kCodeE4m3>(a, p, km, vm, s);
    if (e != cudaSuccess || p.chunks == 1 || p.cluster) return e;
    return run_join<T>(a, s);
}

}  // namespace

extern "C" bfft_status bfft_cache_attention_workspace(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                                      const bfft_attention_desc* d, size_t* bytes) {
    if (!bytes) return fail(BFFT_ERR_VALUE, "null pointer");
    const bfft_status st = check(cache, seqs, d);
    if (st != BFFT_OK) return st;
    if (!seqs->tokens)
        *bytes = 0;
    else
        *bytes = use_tiles(cache, seqs, d) ? plan_tiles(cache, seqs, d, sm_count(d->device)).bytes
                                           : plan_split(cache, seqs, d, sm_count(d->device)).bytes;
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
    Device g(d->device);
    if (!g.ok) return fail(BFFT_ERR_CUDA, "cannot select device %lld", (long long)d->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    a.q_packs = aligned(d->q, 16) && d->q_token % 8 == 0 && d->q_head % 8 == 0;
    a.o_packs = aligned(d->out, 16) && d->o_token % 8 == 0 && d->o_head % 8 == 0;
    unsigned int* status;
    cudaError_t e = device_status_word(&status);
    if (e != cudaSuccess) return launched(e, "cache_attention");
    const bool tiles = use_tiles(cache, seqs, d);
    TilePlan tp{};
    SplitPlan sp{};
    if (tiles)
        tp = plan_tiles(cache, seqs, d, sm_count(d->device));
    else
        sp = plan_split(cache, seqs, d, sm_count(d->device));
    const int chunks = tiles ? tp.chunks : sp.chunks;
    const size_t bytes = tiles ? tp.bytes : sp.bytes;
    if ((tiles ? tp.ctas : sp.ctas) > 0x7fffffffLL || seqs->tokens * d->q_heads > 0x7fffffffLL)
        return fail(BFFT_ERR_SHAPE, "too many rows: %lld", (long long)seqs->tokens);
    if (bytes && (!d->workspace || d->workspace_bytes < (int64_t)bytes))
        return fail(BFFT_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)d->workspace_bytes,
                    (long long)bytes);
    if (bytes && !aligned(d->workspace, 16)) return fail(BFFT_ERR_WORKSPACE, "workspace must be 16-byte aligned");
    float* parts = static_cast<float*>(d->workspace);
    float* stats = parts ? parts + seqs->tokens * d->q_heads * chunks * cache->dim : nullptr;
    count_launches(chunks > 1 && !sp.cluster ? 2 : 1);
    if (tiles) {
        TileArgs ta{a, parts, stats, tp.chunk, tp.chunks, tp.tile_tokens, tp.by_token, tp.slots, status};
        e = d->type == BFFT_F16 ? run_tiles<__half>(ta, tp, cache, s) : run_tiles<__nv_bfloat16>(ta, tp, cache, s);
    } else {
        SplitArgs sa{a, parts, stats, sp.chunk, sp.chunks, sp.tile_tokens, sp.token_tiles, sp.by_token, sp.slots, sp.cluster, sp.entries, status};
        e = d->type == BFFT_F16 ? run_split<__half>(sa, sp, cache, s) : run_split<__nv_bfloat16>(sa, sp, cache, s);
    }
    return launched(e, "cache_attention");
}
