// Norm kernels for rows of __nv_bfloat16.
#include "train_norm.cuh"

namespace lewm {

template cudaError_t launch_norm_rows<__nv_bfloat16>(const NormArgs& p, bool wide, bool backward, int vec, cudaStream_t st);

}  // namespace lewm
