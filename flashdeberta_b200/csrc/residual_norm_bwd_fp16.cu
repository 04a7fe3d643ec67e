// residual_norm's backward over rows of fp16.
#include "residual_norm_bwd.cuh"

namespace fdb {
int norm_bwd_resident_fp16(bool rms, bool post, int mode, bool wide, int threads, int teams) {
  return norm_bwd_resident<__half>(rms, post, mode, wide, threads, teams);
}
int norm_bwd_launch_fp16(const ResidualNormBwdArgs& b, bool wide, cudaStream_t s) { return norm_bwd_launch<__half>(b, wide, s); }
}  // namespace fdb
