// gemm_f16.hip — the matrix product's kernels for f16 operands.
#include "gemm.h"

namespace eas {
template hipError_t gemm_launch_typed<f16>(GemmKernel, const GemmForm&, const GemmParams&, hipStream_t);
template hipError_t gemm_join_typed<f16>(bool, const GemmParams&, hipStream_t);
template hipError_t gemm_pair_typed<f16>(bool, const GemmParams&, const GemmParams&, hipStream_t);
}  // namespace eas
