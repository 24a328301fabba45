// bfft_attention_groups.cu -- the attention kernels for groups of sequences that share a
// prefix.
#include "bfft_attention.cuh"

namespace bfft {

__global__ void __launch_bounds__(kListThreads) k_attention_items(AttentionArgs a, SpanArgs p, ListArgs l) {
    griddep_wait();
    griddep_launch_dependents();
    list_items(a, p, l);
}

BFFT_ATTENTION_FORM(, kGroups)

cudaError_t run_list(const AttentionArgs& a, const SpanArgs& p, const ListArgs& l, cudaStream_t s) {
    return launch_dependent(k_attention_items, 1, kListThreads, 0, s, a, p, l);
}

template cudaError_t run_join_items<__half>(const JoinArgs&, cudaStream_t);
template cudaError_t run_join_items<__nv_bfloat16>(const JoinArgs&, cudaStream_t);

}  // namespace bfft
