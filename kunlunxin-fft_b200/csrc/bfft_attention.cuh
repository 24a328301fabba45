// bfft_attention.cuh -- attention of ragged query rows over a paged 8-bit cache:
// the kernels and their launches.  bfft_attention.cu has the entry points and plans and
// the plain form; bfft_attention_sinks.cu and bfft_attention_groups.cu the other two.
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(t q_i . k_j - m_i),
// over the tokens j that row i sees, with the running maximum m_i and sum kept
// in 32 bits while the tokens pass once.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <type_traits>

#include "../../include/bfft.h"
#include "bfft_async.cuh"
#include "bfft_cache.cuh"
#include "bfft_kernels.cuh"

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

#include "bfft_attention_span.cuh"
#include "bfft_attention_split.cuh"
#include "bfft_attention_tiles.cuh"

namespace bfft {

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

// Defined in bfft_attention.cu: a map of the codes for boxes of 16 tokens.
bool encode_codes(CUtensorMap* m, const void* codes, const bfft_cache_desc* c);
// A map of the queries for boxes of 64 dims, a kv head's heads and a row tile's tokens; false
// where rows and strides do not start on 16 bytes.
bool encode_queries(CUtensorMap* m, const AttentionArgs& a, bool half, int tile_tokens);

template <int DP, typename T, int CODE, int MODE>
cudaError_t launch_tiles(TileArgs a, const TilePlan& p, cudaStream_t s) {
    static std::atomic<bool> ready[64];
    using G = TileGeo<DP>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    auto* kernel = k_attention_tiles<DP, T, CODE, MODE>;
    if (!ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e != cudaSuccess) return e;
        ready[dev].store(true, std::memory_order_release);
    }
    CUtensorMap queries{};
    a.q_tma = encode_queries(&queries, a.a, std::is_same_v<T, __half>, a.tile_tokens);
    return launch_dependent(kernel, (unsigned)p.ctas + (MODE == kGroups && a.others.list != nullptr), G::THREADS, G::SMEM, s, a, queries);
}

template <typename T>
cudaError_t run_join(const SplitArgs& a, cudaStream_t s) {
    const unsigned rows = (unsigned)(a.a.seq.tokens * a.a.q_heads);
    return a.chunks > 16 ? launch_dependent(k_attention_join<T, 16>, rows, 512, 0, s, a)
                         : launch_dependent(k_attention_join<T, 4>, rows, 128, 0, s, a);
}

template <typename T, int MODE>
cudaError_t run_tiles(const TileArgs& a, const TilePlan& p, const bfft_cache_desc* c, cudaStream_t s) {
    cudaError_t e;
    if (c->dim <= 64)
        e = c->code == BFFT_CODE_INT8 ? launch_tiles<64, T, kCodeInt8, MODE>(a, p, s)
                                      : launch_tiles<64, T, kCodeE4m3, MODE>(a, p, s);
    else
        e = c->code == BFFT_CODE_INT8 ? launch_tiles<128, T, kCodeInt8, MODE>(a, p, s)
                                      : launch_tiles<128, T, kCodeE4m3, MODE>(a, p, s);
    if (e != cudaSuccess || MODE == kGroups || p.chunks == 1) return e;
    SplitArgs j{};
    j.a = a.a;
    j.parts = a.parts;
    j.stats = a.stats;
    j.chunks = a.chunks;
    return run_join<T>(j, s);
}

template <int DP, bool EXACT, int NT, typename T, int CODE, int MODE>
cudaError_t launch_split(const SplitArgs& a, const SplitPlan& p, const CUtensorMap& km, const CUtensorMap& vm,
                         cudaStream_t s) {
    static std::atomic<bool> ready[64];
    using G = SplitGeo<DP, EXACT, NT>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    auto* kernel = k_attention_split<DP, EXACT, NT, T, CODE, MODE>;
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

template <typename T, int CODE, int MODE>
cudaError_t split_shape(const SplitArgs& a, const SplitPlan& p, const CUtensorMap& km, const CUtensorMap& vm,
                        cudaStream_t s) {
    const int dim = a.a.cache.dim;
    if (dim == 64)
        return p.nt == 1 ? launch_split<64, true, 1, T, CODE, MODE>(a, p, km, vm, s)
                         : launch_split<64, true, 2, T, CODE, MODE>(a, p, km, vm, s);
    if (dim == 128)
        return p.nt == 1 ? launch_split<128, true, 1, T, CODE, MODE>(a, p, km, vm, s)
                         : launch_split<128, true, 2, T, CODE, MODE>(a, p, km, vm, s);
    if (dim == 256) return launch_split<256, true, 1, T, CODE, MODE>(a, p, km, vm, s);
    if (dim < 128)
        return p.nt == 1 ? launch_split<128, false, 1, T, CODE, MODE>(a, p, km, vm, s)
                         : launch_split<128, false, 2, T, CODE, MODE>(a, p, km, vm, s);
    return launch_split<256, false, 1, T, CODE, MODE>(a, p, km, vm, s);
}

template <typename T, int MODE>
cudaError_t run_split(const SplitArgs& a, const SplitPlan& p, const bfft_cache_desc* c, cudaStream_t s) {
    CUtensorMap km{}, vm{};
    if (c->dim == 64 || c->dim == 128 || c->dim == 256)
        if (!encode_codes(&km, c->k, c) || !encode_codes(&vm, c->v, c)) return cudaErrorNotSupported;
    cudaError_t e = c->code == BFFT_CODE_INT8 ? split_shape<T, kCodeInt8, MODE>(a, p, km, vm, s)
                                              : split_shape<T, kCodeE4m3, MODE>(a, p, km, vm, s);
    if (e != cudaSuccess || MODE == kGroups || p.chunks == 1 || p.cluster) return e;
    return run_join<T>(a, s);
}


// Compiled in bfft_attention_groups.cu.
cudaError_t run_list(const AttentionArgs& a, const SpanArgs& p, const ListArgs& l, cudaStream_t s);

template <typename T>
cudaError_t run_join_items(const JoinArgs& a, cudaStream_t s) {
    const unsigned blocks = (unsigned)(a.a.seq.tokens * a.a.cache.kv_heads);
    const unsigned threads = (a.a.group > kJoinWarps ? 2 : 1) * kJoinWarps * 32;
    if (a.a.cache.dim > 128) return launch_dependent(k_attention_join_items<T, 2, 4>, blocks, threads, 0, s, a);
    return blocks <= 1024 ? launch_dependent(k_attention_join_items<T, 1, 8>, blocks, threads, 0, s, a)
                          : launch_dependent(k_attention_join_items<T, 1, 4>, blocks, threads, 0, s, a);
}

// Compiled in bfft_attention_sinks.cu and bfft_attention_groups.cu.
#define BFFT_ATTENTION_FORM(PREFIX, MODE)                                                                            \
    PREFIX template cudaError_t run_split<__half, MODE>(const SplitArgs&, const SplitPlan&, const bfft_cache_desc*,  \
                                                        cudaStream_t);                                              \
    PREFIX template cudaError_t run_split<__nv_bfloat16, MODE>(const SplitArgs&, const SplitPlan&,                  \
                                                               const bfft_cache_desc*, cudaStream_t);               \
    PREFIX template cudaError_t run_tiles<__half, MODE>(const TileArgs&, const TilePlan&, const bfft_cache_desc*,    \
                                                        cudaStream_t);                                              \
    PREFIX template cudaError_t run_tiles<__nv_bfloat16, MODE>(const TileArgs&, const TilePlan&,                    \
                                                               const bfft_cache_desc*, cudaStream_t);
BFFT_ATTENTION_FORM(extern, kSinks)
BFFT_ATTENTION_FORM(extern, kGroups)
extern template cudaError_t run_join_items<__half>(const JoinArgs&, cudaStream_t);
extern template cudaError_t run_join_items<__nv_bfloat16>(const JoinArgs&, cudaStream_t);

}  // namespace bfft
