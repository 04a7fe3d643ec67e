// residual_norm over rows of fp32.
#include "residual_norm_fwd.cuh"

namespace fdb {
int norm_fwd_launch_fp32(const ResidualNormArgs& a, bool wide, cudaStream_t s) { return norm_fwd_launch<float>(a, wide, s); }
}  // namespace fdb
