// residual_norm over rows of bf16.
#include "residual_norm_fwd.cuh"

namespace fdb {
int norm_fwd_launch_bf16(const ResidualNormArgs& a, bool wide, cudaStream_t s) { return norm_fwd_launch<__nv_bfloat16>(a, wide, s); }
}  // namespace fdb
