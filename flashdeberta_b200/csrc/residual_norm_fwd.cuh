// The forward row kernel of fdb_residual_norm (the mathematics is at the head of residual_norm.cu), for one type of rows per
// translation unit.
#pragma once

#include <algorithm>

#include "internal.h"
#include "launch.h"
#include "residual_norm.h"
#include "row_team.cuh"

namespace fdb {

using ptx::add_f32x2;
using ptx::fma_f32x2;
using ptx::mul_f32x2;

// Up to 1024 elements a row belongs to one warp (ONE): its sums are shuffles, and nothing keeps the next row's loads from starting.
// Longer rows take as many warps, with barriers of their own between them.
constexpr int kNormFwdThreads = 128, kNormFwdWarpElems = 1024;

template <typename T, bool RMS, bool POST, bool WIDE, int V, bool ONE>
__global__ void __launch_bounds__(ONE ? kNormFwdThreads : 256, ONE ? 4 : 2) residual_norm_kernel(const __grid_constant__ ResidualNormArgs a) {
  constexpr int kElems = V * kRowElems;
  __shared__ __align__(16) float s_sums[ONE ? 1 : kNormFwdThreads / 32][TeamSum<1>::kSlots];
  const int team = ONE ? threadIdx.x >> 5 : threadIdx.x / a.team_threads, t = ONE ? threadIdx.x & 31 : threadIdx.x - team * a.team_threads;
  const RowColumns<WIDE, V> cols{t, ONE ? 32 : a.team_threads, a.hidden};
  TeamSum<1> team_sum{s_sums[ONE ? 0 : team], ONE ? 1 : a.team_threads / 32, t >> 5, team + 1, 0};
  if constexpr (!ONE) {
    for (int i = threadIdx.x; i < int(sizeof(s_sums) / sizeof(float)); i += blockDim.x) s_sums[0][i] = 0.f;
    __syncthreads();
  }
  const float inv_hidden = 1.f / (float)a.hidden;
  const T* x = static_cast<const T*>(a.x);
  const T* residual = static_cast<const T*>(a.residual);

  // statistics of a row; afterwards v holds its normalised form
  auto normalise = [&](uint64_t (&v)[kElems / 2], float& mean, float& inv) {
    uint64_t sum = both(0.f);
    float total[1];
    mean = 0.f;
    if constexpr (!RMS) {
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) sum = add_f32x2(sum, v[j]);
      total[0] = fold(sum);
      team_sum(total);
      mean = total[0] * inv_hidden;
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) v[j] = add_f32x2(v[j], cols.inside(j, -mean));
      sum = both(0.f);
    }
#pragma unroll
    for (int j = 0; j < kElems / 2; ++j) sum = fma_f32x2(v[j], v[j], sum);
    total[0] = fold(sum);
    team_sum(total);
    inv = 1.f / sqrtf(fmaf(total[0], inv_hidden, a.eps));
    const uint64_t inv2 = both(inv);
#pragma unroll
    for (int j = 0; j < kElems / 2; ++j) v[j] = mul_f32x2(v[j], inv2);
  };
  auto affine = [&](uint64_t (&v)[kElems / 2], const void* weight, const void* bias) {
    uint64_t p[kElems / 2];
    cols.template load_param<T>(weight, a.param_fp32, 0, p);
    if (!RMS && bias != nullptr) {
      uint64_t q[kElems / 2];
      cols.template load_param<T>(bias, a.param_fp32, 0, q);
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) v[j] = fma_f32x2(v[j], p[j], q[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) v[j] = mul_f32x2(v[j], p[j]);
    }
  };

  const int64_t row = (int64_t)blockIdx.x * a.teams + team;
  if (row >= a.rows) return;
  const int64_t at = row * a.hidden;
  RowWords<T, V> rx, rr;
  cols.load(x + at, rx);
  if (residual != nullptr) cols.load(residual + at, rr);
  uint64_t v[kElems / 2], p[kElems / 2];
  float4 stats = make_float4(0.f, 1.f, 0.f, 1.f);
  unpack(rx, v);
  if constexpr (POST) {
    normalise(v, stats.x, stats.y);
    affine(v, a.post_weight, a.post_bias);
  }
  if (a.gate != nullptr) {
    cols.template load_param<T>(a.gate, a.gate_fp32, (int64_t)((uint32_t)row / a.gate_rows) * a.hidden, p);
#pragma unroll
    for (int j = 0; j < kElems / 2; ++j) v[j] = mul_f32x2(v[j], p[j]);
  }
  if (residual != nullptr) {
    const uint64_t scale = both(a.residual_scale);
    unpack(rr, p);
#pragma unroll
    for (int j = 0; j < kElems / 2; ++j) v[j] = fma_f32x2(scale, p[j], v[j]);
  }
  if (a.stream != nullptr) cols.store(static_cast<T*>(a.stream) + at, v);
  normalise(v, stats.z, stats.w);
  affine(v, a.weight, a.bias);
  cols.store(static_cast<T*>(a.normed) + at, v);
  if (a.stats != nullptr && t == 0) a.stats[row] = stats;
}

template <typename T, bool RMS, bool POST, bool WIDE, int V, bool ONE>
int norm_fwd_launch_kernel(const ResidualNormArgs& a, cudaStream_t s) {
  const int threads = a.teams * a.team_threads;
  residual_norm_kernel<T, RMS, POST, WIDE, V, ONE><<<(unsigned)((a.rows + a.teams - 1) / a.teams), (unsigned)threads, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "residual_norm launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

// Warps of a row, elements per thread and rows per CTA from the width.
template <typename T> int norm_fwd_launch(ResidualNormArgs a, bool wide, cudaStream_t s) {
  const int warps = (a.hidden + kNormFwdWarpElems - 1) / kNormFwdWarpElems;
  const int v = (a.hidden + warps * 32 * kRowElems - 1) / (warps * 32 * kRowElems);
  a.team_threads = warps * 32;
  a.teams = std::max(1, kNormFwdThreads / a.team_threads);
#define FDB_FWD4(R, P, W, V, ONE) norm_fwd_launch_kernel<T, R, P, W, V, ONE>(a, s)
#define FDB_FWD3(R, P, W)                                                                  \
  (warps > 1 ? (v == 3 ? FDB_FWD4(R, P, W, 3, false) : FDB_FWD4(R, P, W, 4, false))       \
             : (v == 1 ? FDB_FWD4(R, P, W, 1, true)                                        \
                       : (v == 2 ? FDB_FWD4(R, P, W, 2, true) : (v == 3 ? FDB_FWD4(R, P, W, 3, true) : FDB_FWD4(R, P, W, 4, true)))))
#define FDB_FWD2(R, P) (wide ? FDB_FWD3(R, P, true) : FDB_FWD3(R, P, false))
  const bool post = a.post_weight != nullptr;
  if (a.rms) return post ? FDB_FWD2(true, true) : FDB_FWD2(true, false);
  return post ? FDB_FWD2(false, true) : FDB_FWD2(false, false);
#undef FDB_FWD4
#undef FDB_FWD3
#undef FDB_FWD2
}

}  // namespace fdb
