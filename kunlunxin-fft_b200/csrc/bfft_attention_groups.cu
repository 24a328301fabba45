// bfft_attention_groups.cu -- the attention kernels for groups of sequences that share a
// prefix.
#include "bfft_attention.cuh"

namespace bfft {

BFFT_ATTENTION_FORM(, kGroups)
template cudaError_t run_join_items<__half>(const JoinArgs&, cudaStream_t);
template cudaError_t run_join_items<__nv_bfloat16>(const JoinArgs&, cudaStream_t);

}  // namespace bfft
