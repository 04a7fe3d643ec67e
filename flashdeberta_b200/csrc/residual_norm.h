// What the kernels of residual_norm.cu and residual_norm_bwd.cuh take.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace fdb {

struct ResidualNormArgs {
  const void *x, *residual, *weight, *bias, *post_weight, *post_bias, *gate;
  void *normed, *stream;
  float4* stats;       // per row: mean and inverse deviation of x, of the stream
  int64_t rows;
  uint32_t gate_rows;  // rows that share a row of the gate
  int hidden, team_threads, teams;
  float residual_scale, eps;
  bool rms, param_fp32, gate_fp32;
};

// One gate row (or no gate) for all rows; one for each of several groups of rows; one for each row.
enum : int { kGateChannel = 0, kGateGroups = 1, kGateElement = 2 };

struct ResidualNormBwdArgs {
  ResidualNormArgs f;
  const void *dnormed, *dstream;
  void *dx, *dresidual, *dweight, *dbias, *dpost_weight, *dpost_bias, *dgate;
  float* parts;        // (ctas, vectors, hidden): each CTA's sums over its rows
  float* slots;        // (workers + groups, 2, hidden): A and B of a worker's rows in a group
  int64_t workers;     // teams that have rows: worker w the rows [rows w / workers, rows (w + 1) / workers)
  int ctas, vectors, mode, groups;
  int ring_at;         // where in shared memory rows lie that are on their way
};

constexpr int kNormBwdThreads = 512;  // threads of a backward CTA whose rows take fewer: one CTA per SM, of several rows at a time

// the worker that has a row
__host__ __device__ inline int64_t residual_norm_worker_of(int64_t row, int64_t rows, int64_t workers) { return ((row + 1) * workers - 1) / rows; }

// The row kernels, per type of rows.
#define FDB_NORM(TYPE)                                                                \
  int norm_fwd_launch_##TYPE(const ResidualNormArgs& a, bool wide, cudaStream_t s);   \
  int norm_bwd_launch_##TYPE(const ResidualNormBwdArgs& b, bool wide, cudaStream_t s);
FDB_NORM(bf16)
FDB_NORM(fp16)
FDB_NORM(fp32)
#undef FDB_NORM

}  // namespace fdb
