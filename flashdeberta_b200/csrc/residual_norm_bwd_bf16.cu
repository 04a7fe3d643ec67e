// residual_norm's backward over rows of bf16.
#include "residual_norm_bwd.cuh"

namespace fdb {
int norm_bwd_launch_bf16(const ResidualNormBwdArgs& b, bool wide, cudaStream_t s) { return norm_bwd_launch<__nv_bfloat16>(b, wide, s); }
}  // namespace fdb
