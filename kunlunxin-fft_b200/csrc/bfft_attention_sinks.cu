// bfft_attention_sinks.cu -- the attention kernels for windows beside which first tokens
// stay visible.
#include "bfft_attention.cuh"

namespace bfft {

BFFT_ATTENTION_FORM(, kSinks)

}  // namespace bfft
