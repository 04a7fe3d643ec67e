// residual_norm's backward over rows of fp16.
#include "residual_norm_bwd.cuh"

namespace fdb {
int norm_bwd_launch_fp16(const ResidualNormBwdArgs& b, bool wide, cudaStream_t s) { return norm_bwd_launch<__half>(b, wide, s); }
}  // namespace fdb
