// bfft_attention_groups.cu -- the attention kernels for groups of sequences that share a
// prefix.
#include "bfft_attention.cuh"

namespace bfft {

// Lists the items of more units: one block, long pieces before short ones (in sixteen
// classes), as blocks start in the order of their items.  The order within a class is that
// of the atomics; a token's parts are joined in the order of its axis wherever they lie.
constexpr int kListThreads = 512;
__global__ void __launch_bounds__(kListThreads) k_attention_items(AttentionArgs a, SpanArgs p, ItemArgs x, int tile,
                                                                  int parts, Item* list, int* count) {
    constexpr int WARPS = kListThreads / 32, CLASSES = 16;
    __shared__ float sums[WARPS];
    __shared__ int first[CLASSES];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int groups = x.prefixes ? p.n_groups : 0, units = unit_count(p, x, a.seq.seqs);
    if (tid < CLASSES) first[tid] = 0;
    float total = 0.f;
    unsigned chunk = 1;
    // three looks at every unit: the sum, the classes' counts, the items
#pragma unroll 1
    for (int look = 0; look < 3; ++look) {
#pragma unroll 1
        for (int u = tid; u < units; u += kListThreads) {
            const Unit v = unit_of(a, p, x, u, tile, parts);
            if (look == 0) {
                total += (float)v.tiles * (float)v.length;
                continue;
            }
            const int pieces = pieces_of(v, chunk), mine = v.tiles * pieces;
            const unsigned each = ((unsigned)v.length + pieces - 1) / pieces;
            const int of = CLASSES - 1 - (int)min(each * (float)CLASSES / (float)chunk, CLASSES - 1.f);
            const int at = mine ? atomicAdd(&first[of], mine) : 0;
            if (look == 2)
                for (int k = 0; k < mine && at + k < x.most; ++k)
                    fill_item(list[at + k], v, u < groups, k, pieces, tile, parts);
        }
        if (look == 0) {
#pragma unroll
            for (int w = 16; w; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
            if (lane == 0) sums[warp] = total;
            __syncthreads();
            total = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) total += sums[w];
            chunk = item_tokens(x, total);
        } else if (look == 1) {
            __syncthreads();
            if (tid == 0) {
                int sum = 0;
                for (int c = 0; c < CLASSES; ++c) {
                    const int n = first[c];
                    first[c] = sum;
                    sum += n;
                }
                *count = sum < x.most ? sum : (int)x.most;
            }
            __syncthreads();
        }
    }
}

BFFT_ATTENTION_FORM(, kGroups)

cudaError_t list_items(const AttentionArgs& a, const SpanArgs& p, const ItemArgs& x, int tile, int parts, Item* list,
                       int* count, cudaStream_t s) {
    return launch_dependent(k_attention_items, 1, kListThreads, 0, s, a, p, x, tile, parts, list, count);
}

template cudaError_t run_join_items<__half>(const JoinArgs&, cudaStream_t);
template cudaError_t run_join_items<__nv_bfloat16>(const JoinArgs&, cudaStream_t);

}  // namespace bfft
