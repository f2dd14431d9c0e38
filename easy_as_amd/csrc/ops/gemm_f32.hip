// gemm_f32.hip — the matrix product's kernels for f32 operands.
#include "gemm.h"

namespace eas {
template hipError_t gemm_launch_typed<float>(GemmKernel, const GemmForm&, const GemmParams&, hipStream_t);
template hipError_t gemm_join_typed<float>(bool, const GemmParams&, hipStream_t);
template hipError_t gemm_pair_typed<float>(bool, const GemmParams&, const GemmParams&, hipStream_t);
}  // namespace eas
