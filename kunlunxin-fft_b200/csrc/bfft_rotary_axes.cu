// bfft_rotary_axes.cu -- the rotation and the append for positions of several axes
// (see bfft_rotary.cuh); their entry points are in bfft_rotary.cu.
#include "bfft_rotary.cuh"

namespace bfft {

template cudaError_t launch_rotate(int64_t, int, int, const RotateArgs&, const AxisMap&, dim3, dim3, cudaStream_t);
template cudaError_t launch_append(int64_t, int, int, int, const AppendArgs&, const AxisMap&, const AppendPlan&, cudaStream_t);

}  // namespace bfft
