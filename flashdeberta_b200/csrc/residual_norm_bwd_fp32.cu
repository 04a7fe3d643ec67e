// residual_norm's backward over rows of fp32.
#include "residual_norm_bwd.cuh"

namespace fdb {
int norm_bwd_launch_fp32(const ResidualNormBwdArgs& b, bool wide, cudaStream_t s) { return norm_bwd_launch<float>(b, wide, s); }
}  // namespace fdb
