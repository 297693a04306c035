// Norm kernels for rows of __half.
#include "train_norm.cuh"

namespace lewm {

template cudaError_t launch_norm_rows<__half>(const NormArgs& p, bool wide, bool backward, int vec, cudaStream_t st);

}  // namespace lewm
