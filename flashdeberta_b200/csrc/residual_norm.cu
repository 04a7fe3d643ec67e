// stream = residual_scale * residual + gate (.) Norm_post(x),  normed = Norm(stream): what lies between two blocks of a layer,
// in one pass over the rows, and its backward.  Norm is LayerNorm or RMSNorm; Norm_post and the gate may be absent.
//
// Forward (residual_norm_fwd.cuh).  With one row in the registers of a warp or several (row_team.cuh) both norms are sums over the
// team: mean, then centred squares (two passes over registers: rows whose mean is far from zero lose nothing).  Sums in fp32, `normed`
// from the sum before it is rounded to the rows' type.  HBM-bound: x and residual read, both results written.  Measured (four sets of
// inputs in turn, of the copy bandwidth of 6548 GB/s): 16384 x 1024 bf16, one LayerNorm 20.7 us = 99 %, RMS norms on both sides and a
// gate 23.8 us = 86 %, LayerNorms on both sides 28 us = 73 % (four sums one after another, 16 rows on an SM), 65536 x 256
// 30 us = 68 %, one LayerNorm 21 us = 97 %; 8192 x 1024 fp32 21.7 us = 94 %; rows of several warps 55 to 71 %; 16-bit rows that start anywhere 30 %.
//
// Backward (residual_norm_bwd.cuh), for every row with the statistics that the forward kept (mean and inverse deviation of both norms):
//     dz = dstream + inv2 (y - mean(y) - zhat mean(y zhat)),   y = weight dnormed,  zhat = (stream - mean2) inv2
//     dresidual = residual_scale dz,   du = gate dz,
//     dx = inv1 (p - mean(p) - xhat mean(p xhat)),             p = post_weight du,  xhat = (x - mean1) inv1
// (RMSNorm without the mean terms).  The stream is computed again from x and residual, in fp32 as the forward had it: the rounded one
// would cost as many bytes and put its rounding into zhat.  HBM-bound by its bytes (four tensors of rows read, two written), in fact by
// its instructions, some 45 per element, and the chain of two sums a row on 16 warps per SM: 32768 x 1024 bf16 81 us = 76 % with one
// LayerNorm, 92 us = 67 % with RMS norms on both sides and a gate per sequence, 101 us = 61 % with LayerNorms; above 4096 columns a
// CTA of 1024 threads has too few registers (232 us at 4096 x 8192).  On the way (32768 x 1024, RMS norms): sums through a loop over
// the warps and parameters loaded for every row 125 us; parameters in shared memory 107; two-wide arithmetic 92 to 95; with
// LayerNorms 114, and 101 once rows waited in shared memory.
//
// Sums over rows (gradients of weights, biases and gate) stay in registers while a thread walks its rows, one per column and sum;
// they go to memory once per CTA and a second kernel adds them up in a fixed order: no atomics, the same bits every time.
// With A = sum dz xhat and B = sum dz over the rows that share a gate row, the three gradients of that stage are
//     dpost_weight = sum gate A,   dpost_bias = sum gate B,   dgate = post_weight A + post_bias B
// so a gate per channel takes no sums of its own.  With a gate per group of rows a worker's rows are one range; A and B leave
// the registers whenever a group ends, to slot (worker + group), which no two pairs share because both only grow along the rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "internal.h"
#include "launch.h"
#include "residual_norm.h"
#include "row_team.cuh"

namespace fdb {
namespace {

unsigned type_bytes(int dtype) { return dtype == FDB_FP32 ? 4u : 2u; }

// Checks of a call and its kernel arguments; `wide`: rows and vectors may be read eight elements at a time.
int prepare(const fdb_residual_norm_params* p, ResidualNormArgs* a, bool* wide) {
  if (p == nullptr || p->struct_bytes != sizeof(fdb_residual_norm_params))
    return fail(FDB_ERR_INVALID_ARGUMENT, "fdb_residual_norm_params: NULL or struct_bytes %u != %zu", p ? p->struct_bytes : 0u,
                sizeof(fdb_residual_norm_params));
  if (p->dtype != FDB_BF16 && p->dtype != FDB_FP16 && p->dtype != FDB_FP32)
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: dtype %d", p->dtype);
  if ((p->param_dtype != p->dtype && p->param_dtype != FDB_FP32) || (p->gate != nullptr && p->gate_dtype != p->dtype && p->gate_dtype != FDB_FP32))
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: parameters are of the rows' type or fp32");
  if (p->rows < 0 || p->hidden <= 0) return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: rows %lld, hidden %d", (long long)p->rows, p->hidden);
  if (p->rows > 2147483647LL || p->hidden > kRowHiddenMax)
    return fail(FDB_ERR_LIMIT, "residual_norm: %lld rows of %d; at most 2^31 - 1 rows of %d", (long long)p->rows, p->hidden, kRowHiddenMax);
  if (p->x == nullptr || p->weight == nullptr || p->normed == nullptr)
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: x, weight and normed must not be NULL");
  if (p->rms != 0 && (p->bias != nullptr || p->post_bias != nullptr))
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: the RMS norm takes no bias");
  if (p->post_bias != nullptr && p->post_weight == nullptr) return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: post_bias without post_weight");
  if (p->gate != nullptr && (p->gate_rows <= 0 || p->gate_rows > 2147483647LL || p->rows % p->gate_rows != 0))
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm: %lld rows, %lld of them per row of the gate", (long long)p->rows, (long long)p->gate_rows);
  const unsigned size = type_bytes(p->dtype), param = type_bytes(p->param_dtype), gate = type_bytes(p->gate_dtype);
  if (!aligned_to(size, p->x, p->residual, p->normed, p->stream) || !aligned_to(param, p->weight, p->bias, p->post_weight, p->post_bias) ||
      (p->gate != nullptr && !aligned_to(gate, p->gate)) || !aligned_to(16, p->stats))
    return fail(FDB_ERR_ALIGNMENT, "residual_norm: tensors must be aligned to their elements, stats to 16 bytes");
  *wide = p->hidden % kRowElems == 0 && aligned_to(8 * size, p->x, p->residual, p->normed, p->stream) &&
          aligned_to(8 * param, p->weight, p->bias, p->post_weight, p->post_bias) && (p->gate == nullptr || aligned_to(8 * gate, p->gate));
  a->x = p->x; a->residual = p->residual;
  a->weight = p->weight; a->bias = p->bias; a->post_weight = p->post_weight; a->post_bias = p->post_bias; a->gate = p->gate;
  a->normed = p->normed; a->stream = p->stream; a->stats = reinterpret_cast<float4*>(p->stats);
  a->rows = p->rows; a->gate_rows = p->gate != nullptr ? (uint32_t)p->gate_rows : 1u;
  a->hidden = p->hidden;
  a->residual_scale = p->residual_scale; a->eps = p->eps;
  a->rms = p->rms != 0; a->param_fp32 = p->param_dtype == FDB_FP32; a->gate_fp32 = p->gate_dtype == FDB_FP32;
  a->team_threads = a->teams = 0;
  return FDB_OK;
}

// How the gate's rows are shared (without rows there are none, and nothing is shared).
int gate_mode(const fdb_residual_norm_params& p) {
  if (p.gate == nullptr || p.gate_rows == p.rows) return kGateChannel;
  return p.gate_rows == 1 || p.rows == 0 ? kGateElement : kGateGroups;
}

// Teams, CTAs and workspace of a backward call.
void plan(const fdb_residual_norm_params& p, ResidualNormBwdArgs* b, uint64_t* bytes) {
  const int mode = gate_mode(p);
  b->f.team_threads = row_team_threads(p.hidden);
  b->f.teams = std::max(1, kNormBwdThreads / b->f.team_threads);
  const int64_t want = (p.rows + b->f.teams - 1) / b->f.teams;
  b->ctas = (int)std::max<int64_t>(1, std::min<int64_t>(want, std::max(1, sm_count())));
  b->workers = std::min((int64_t)b->ctas * b->f.teams, p.rows);  // each has a row
  b->vectors = (p.rms != 0 ? 1 : 2) * 2;  // of weight and bias, and A and B or what they become
  b->groups = mode == kGateGroups ? (int)(p.rows / p.gate_rows) : 0;
  const uint64_t row = uint64_t(p.hidden) * sizeof(float);
  *bytes = uint64_t(b->ctas) * b->vectors * row + (b->groups > 0 ? (uint64_t(b->workers) + b->groups) * 2 * row : 0);
}

}  // namespace

// ---- sums over rows: from the CTAs' parts to gradients -----------------------------------------------------------------------------
namespace {

constexpr int kFinishCols = 32, kFinishRows = 16;

// One thread's column of a sum over `n` rows `stride` floats apart, the thread's share of the rows in order; then the shares, in order.
__device__ __forceinline__ float column_total(const float* p, int n, int64_t stride, float (*share)[kFinishCols + 1], bool live) {
  float sum = 0.f;
  if (live) {
#pragma unroll 4
    for (int i = threadIdx.y; i < n; i += kFinishRows) sum += p[i * stride];
  }
  __syncthreads();
  share[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int y = 0; y < kFinishRows; ++y) sum += share[y][threadIdx.x];
  return sum;
}

template <typename T> __device__ __forceinline__ float param_at(const void* p, bool fp32, int64_t i) {
  return fp32 ? static_cast<const float*>(p)[i] : to_float<T>(static_cast<const T*>(p)[i]);
}
template <typename T> __device__ __forceinline__ void put_param(void* p, bool fp32, int64_t i, float v) {
  if (fp32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = from_float<T>(v);
}

template <typename T>
__global__ void __launch_bounds__(kFinishCols * kFinishRows) residual_norm_sums_kernel(const __grid_constant__ ResidualNormBwdArgs b) {
  __shared__ float share[kFinishRows][kFinishCols + 1];
  const ResidualNormArgs& f = b.f;
  const int c = blockIdx.x * kFinishCols + threadIdx.x;
  const bool live = c < f.hidden, writes = live && threadIdx.y == 0;
  const int cc = live ? c : 0;
  const bool post = f.post_weight != nullptr;
  ptx::grid_wait();
  if (blockIdx.y == 0) {  // sums over all rows
    const int64_t stride = (int64_t)b.vectors * f.hidden;
    const int per_norm = b.vectors / 2;
    const float* part = b.parts + cc;
    if (b.dweight != nullptr) {
      const float v = column_total(part, b.ctas, stride, share, live);
      if (writes) put_param<T>(b.dweight, f.param_fp32, c, v);
    }
    if (b.dbias != nullptr) {
      const float v = column_total(part + f.hidden, b.ctas, stride, share, live);
      if (writes) put_param<T>(b.dbias, f.param_fp32, c, v);
    }
    const bool channel = b.mode == kGateChannel && f.gate != nullptr;
    if (b.dpost_weight == nullptr && b.dpost_bias == nullptr && !(channel && b.dgate != nullptr)) return;
    const float sum_a = column_total(part + (int64_t)per_norm * f.hidden, b.ctas, stride, share, live);
    const float sum_b = per_norm == 2 ? column_total(part + 3ll * f.hidden, b.ctas, stride, share, live) : 0.f;
    if (!writes) return;
    const float gate = channel ? param_at<T>(f.gate, f.gate_fp32, c) : 1.f;
    if (b.dpost_weight != nullptr) put_param<T>(b.dpost_weight, f.param_fp32, c, gate * sum_a);
    if (b.dpost_bias != nullptr) put_param<T>(b.dpost_bias, f.param_fp32, c, gate * sum_b);
    if (channel && b.dgate != nullptr) {
      float v = sum_a;
      if (post) {
        v = param_at<T>(f.post_weight, f.param_fp32, c) * sum_a;
        if (f.post_bias != nullptr) v = fmaf(param_at<T>(f.post_bias, f.param_fp32, c), sum_b, v);
      }
      put_param<T>(b.dgate, f.gate_fp32, c, v);
    }
    return;
  }
  // the gate's gradient of one group after another: the slots of the workers that share its rows
  for (int64_t g = (int64_t)blockIdx.y - 1; g < b.groups; g += (int64_t)gridDim.y - 1) {
    const int64_t first = residual_norm_worker_of(g * f.gate_rows, f.rows, b.workers);
    const int64_t last = residual_norm_worker_of((g + 1) * f.gate_rows - 1, f.rows, b.workers);
    const float* slot = b.slots + (first + g) * 2 * f.hidden + cc;
    const int n = (int)(last - first + 1);
    float v = column_total(slot, n, 2ll * f.hidden, share, live);
    if (post) {
      const float sum_b = f.post_bias != nullptr ? column_total(slot + f.hidden, n, 2ll * f.hidden, share, live) : 0.f;
      if (live) {
        v *= param_at<T>(f.post_weight, f.param_fp32, c);
        if (f.post_bias != nullptr) v = fmaf(param_at<T>(f.post_bias, f.param_fp32, c), sum_b, v);
      }
    }
    if (writes) put_param<T>(b.dgate, f.gate_fp32, g * f.hidden + c, v);
  }
}

}  // namespace
}  // namespace fdb

using namespace fdb;

extern "C" FDB_API int fdb_residual_norm(const fdb_residual_norm_params* p, void* stream) {
  clear_error();
  ResidualNormArgs a;
  bool wide;
  const int rc = prepare(p, &a, &wide);
  if (rc != FDB_OK) return rc;
  if (p->rows == 0) return FDB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->dtype == FDB_BF16) return norm_fwd_launch_bf16(a, wide, s);
  return p->dtype == FDB_FP16 ? norm_fwd_launch_fp16(a, wide, s) : norm_fwd_launch_fp32(a, wide, s);
}

namespace {
int prepare_bwd(const fdb_residual_norm_bwd_params* p, ResidualNormBwdArgs* b, bool* wide, uint64_t* bytes) {
  if (p == nullptr || p->struct_bytes != sizeof(fdb_residual_norm_bwd_params))
    return fail(FDB_ERR_INVALID_ARGUMENT, "fdb_residual_norm_bwd_params: NULL or struct_bytes %u != %zu", p ? p->struct_bytes : 0u,
                sizeof(fdb_residual_norm_bwd_params));
  int rc = prepare(&p->fwd, &b->f, wide);
  if (rc != FDB_OK) return rc;
  const fdb_residual_norm_params& f = p->fwd;
  if (f.stats == nullptr || (p->dnormed == nullptr && p->dstream == nullptr) || p->dx == nullptr)
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm backward: stats, dx and one of dnormed and dstream must not be NULL");
  if ((p->dresidual != nullptr && f.residual == nullptr) || (p->dbias != nullptr && f.bias == nullptr) ||
      (p->dpost_weight != nullptr && f.post_weight == nullptr) || (p->dpost_bias != nullptr && f.post_bias == nullptr) ||
      (p->dgate != nullptr && f.gate == nullptr))
    return fail(FDB_ERR_INVALID_ARGUMENT, "residual_norm backward: a gradient of a tensor that the forward did not have");
  const unsigned size = f.dtype == FDB_FP32 ? 4u : 2u, param = f.param_dtype == FDB_FP32 ? 4u : 2u, gate = f.gate_dtype == FDB_FP32 ? 4u : 2u;
  if (!aligned_to(size, p->dnormed, p->dstream, p->dx, p->dresidual) || !aligned_to(param, p->dweight, p->dbias, p->dpost_weight, p->dpost_bias) ||
      (p->dgate != nullptr && !aligned_to(gate, p->dgate)))
    return fail(FDB_ERR_ALIGNMENT, "residual_norm backward: tensors must be aligned to their elements");
  *wide = *wide && aligned_to(8 * size, p->dnormed, p->dstream, p->dx, p->dresidual) && (p->dgate == nullptr || aligned_to(8 * gate, p->dgate)) &&
          aligned_to(32, p->workspace);
  b->dnormed = p->dnormed; b->dstream = p->dstream; b->dx = p->dx; b->dresidual = p->dresidual;
  b->dweight = p->dweight; b->dbias = p->dbias; b->dpost_weight = p->dpost_weight; b->dpost_bias = p->dpost_bias; b->dgate = p->dgate;
  b->mode = gate_mode(f);
  plan(f, b, bytes);
  return FDB_OK;
}
}  // namespace

extern "C" FDB_API uint64_t fdb_residual_norm_bwd_workspace_bytes(const fdb_residual_norm_bwd_params* p) {
  clear_error();
  ResidualNormBwdArgs b;
  bool wide;
  uint64_t bytes = 0;
  return prepare_bwd(p, &b, &wide, &bytes) == FDB_OK ? bytes : 0;
}

extern "C" FDB_API int fdb_residual_norm_bwd(const fdb_residual_norm_bwd_params* p, void* stream) {
  clear_error();
  ResidualNormBwdArgs b;
  bool wide;
  uint64_t bytes = 0;
  int rc = prepare_bwd(p, &b, &wide, &bytes);
  if (rc != FDB_OK) return rc;
  if (p->workspace == nullptr || p->workspace_bytes < bytes || !aligned_to(32, p->workspace))
    return fail(FDB_ERR_WORKSPACE, "residual_norm backward: workspace of %llu bytes needed (32-byte aligned), %llu given",
                (unsigned long long)bytes, (unsigned long long)p->workspace_bytes);
  b.parts = static_cast<float*>(p->workspace);
  b.slots = b.parts + (int64_t)b.ctas * b.vectors * b.f.hidden;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // (without rows the CTA that is launched has none either: it leaves sums of zero)
  auto launch_rows = p->fwd.dtype == FDB_BF16 ? norm_bwd_launch_bf16 : (p->fwd.dtype == FDB_FP16 ? norm_bwd_launch_fp16 : norm_bwd_launch_fp32);
  if ((rc = launch_rows(b, wide, s)) != FDB_OK) return rc;
  const bool group_gate = b.groups > 0 && b.dgate != nullptr;
  if (b.dweight == nullptr && b.dbias == nullptr && b.dpost_weight == nullptr && b.dpost_bias == nullptr && (b.dgate == nullptr || b.mode == kGateElement))
    return FDB_OK;
  const dim3 grid((unsigned)((b.f.hidden + kFinishCols - 1) / kFinishCols), (unsigned)(1 + (group_gate ? std::min(b.groups, 1024) : 0)));
  auto kernel = p->fwd.dtype == FDB_BF16 ? residual_norm_sums_kernel<__nv_bfloat16>
                                          : (p->fwd.dtype == FDB_FP16 ? residual_norm_sums_kernel<__half> : residual_norm_sums_kernel<float>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kFinishCols, kFinishRows);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  void* args[] = {&b};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), args);
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "residual_norm sums launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}
