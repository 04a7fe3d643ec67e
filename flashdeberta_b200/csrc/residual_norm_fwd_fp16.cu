// residual_norm over rows of fp16.
#include "residual_norm_fwd.cuh"

namespace fdb {
int norm_fwd_launch_fp16(const ResidualNormArgs& a, bool wide, cudaStream_t s) { return norm_fwd_launch<__half>(a, wide, s); }
}  // namespace fdb
