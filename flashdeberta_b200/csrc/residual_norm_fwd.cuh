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
// Longer rows take as many warps, with barriers of their own between them.  A CTA stays and takes row after row: weights and biases
// (and a channel's gate) are converted to fp32 once, into shared memory, and the next rows are on their way while one is worked on.
constexpr int kNormFwdWarpElems = 1024;
constexpr int kNormFwdThreads = 512;  // of a CTA of longer rows, one per SM (at most 128 registers a thread)
// Whether 16-bit rows of one warp are on their way in shared memory, two ahead, instead of one ahead in registers.  16 M elements in bf16,
// registers against shared memory, without a gate, one per channel, per sequence, per element:
//    256 columns, LayerNorms on both sides  34.9 35.5 39.2 41.0 and 29.3 30.8 33.7 36.5    one LayerNorm  26.7 27.4 31.5 33.9 and 26.6 26.7 27.1 31.0 us
//    512                                    29.1 30.8 33.0 35.0     27.4 29.5 30.8 32.8                   26.5 26.8 28.0 32.3     25.9 26.4 25.8 30.5
//    768                                    27.0 27.1 30.9 34.0     26.9 28.9 31.1 34.4                   25.9 26.5 27.4 31.0     26.4 26.7 27.0 31.0
//   1024                                    30.7 31.9 32.7 36.9     27.6 30.0 32.1 34.0                   25.8 26.6 26.3 30.9     25.7 26.4 27.3 31.0
// RMS norms gain at 256 and 512 (both sides 30.8 and 26.8, 27.2 and 25.6) and are even at 768 and 1024.  Only both LayerNorms at 768 with a gate
// per channel lose (27.1 and 28.9); the gate is no part of the rule, which would take another set of kernels for that one form.
constexpr int kNormFwdRows = 2;
template <typename T> __host__ __device__ constexpr bool norm_fwd_ring(bool rms, bool post, bool wide, int v, bool one) {
  return sizeof(T) == 2 && wide && one && (v < 4 || (post && !rms));
}
// CTAs per SM of rows of one warp, 4 rows each: what the registers of V x 8 elements per thread allow.
constexpr int norm_fwd_ctas(int v, bool ring) { return v == 1 ? 10 : (v == 2 ? 7 : (v == 3 && ring ? 5 : 4)); }

template <typename T, bool RMS, bool POST, bool WIDE, int V, bool ONE>
__global__ void __launch_bounds__(ONE ? 128 : kNormFwdThreads, ONE ? norm_fwd_ctas(V, norm_fwd_ring<T>(RMS, POST, WIDE, V, ONE)) : 1)
    residual_norm_kernel(const __grid_constant__ ResidualNormArgs a) {
  constexpr int kElems = V * kRowElems, kPairs = kElems / 2;
  extern __shared__ __align__(16) float4 s_vectors[];
  __shared__ __align__(16) float s_sums[ONE ? 1 : kNormFwdThreads / 64][TeamSum<1>::kSlots];
  const int threads = ONE ? 32 : a.team_threads;
  const int team = ONE ? threadIdx.x >> 5 : threadIdx.x / threads, t = ONE ? threadIdx.x & 31 : threadIdx.x - team * threads;
  const RowColumns<row_mode<T>(WIDE), V> cols{t, threads, a.hidden};
  TeamSum<1> team_sum{s_sums[ONE ? 0 : team], threads / 32, t >> 5, team + 1, 0};
  const float inv_hidden = 1.f / (float)a.hidden;

  RowWords<T, V> rx, rr, nx, nr;
  auto fetch = [&](int64_t row, RowWords<T, V>& wx, RowWords<T, V>& wr) {
    cols.load(static_cast<const T*>(a.x) + row * a.hidden, wx);
    if (a.residual != nullptr) cols.load(static_cast<const T*>(a.residual) + row * a.hidden, wr);
  };
  const int64_t step = (int64_t)gridDim.x * a.teams;
  int64_t row = (int64_t)blockIdx.x * a.teams + team;
  constexpr bool kRing = norm_fwd_ring<T>(RMS, POST, WIDE, V, ONE);
  constexpr bool kAhead = sizeof(T) == 2 && WIDE && !kRing;  // (fp32 rows would take too many registers, single elements and shifted pieces are put into words at once)
  if (kAhead && row < a.rows) fetch(row, nx, nr);
  // rows on their way in shared memory: each thread copies what it reads itself, so it waits for its own copies alone
  uint4* s_ring = reinterpret_cast<uint4*>(s_vectors + 5 * (kElems / 4) * threads) + threadIdx.x;
  auto send = [&](int64_t r, int slot) {
    if (r < a.rows) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!cols.live(i * kRowElems)) continue;
        const int64_t from = r * a.hidden + cols.col(i * kRowElems);
        ptx::copy_async_16B(ptx::smem_u32(s_ring + (slot * 2 * V + i) * 128), static_cast<const T*>(a.x) + from);
        if (a.residual != nullptr) ptx::copy_async_16B(ptx::smem_u32(s_ring + (slot * 2 * V + V + i) * 128), static_cast<const T*>(a.residual) + from);
      }
    }
    ptx::copy_async_commit();
  };
  int slot = 0;
  if constexpr (kRing) {
#pragma unroll
    for (int i = 0; i < V; ++i)  // what lies behind the end of the row reads as zeros all the time
      if (!cols.live(i * kRowElems))
        for (int k = 0; k < 2 * kNormFwdRows; ++k) s_ring[(k * V + i) * 128] = make_uint4(0, 0, 0, 0);
    for (int k = 0; k < kNormFwdRows; ++k) send(row + k * step, k);
  }

  // vectors over the columns: 16-byte pieces, each piece of the team's threads side by side
  enum : int { kWeight = 0, kBias = 1, kPostWeight = 2, kPostBias = 3, kGateVector = 4 };
  const bool channel_gate = a.gate != nullptr && a.gate_rows == a.rows;
  auto put_vector = [&](int v, const void* p, bool fp32) {
    float q[kElems];
    if (p != nullptr) cols.template load_param<T>(p, fp32, 0, q);
    else
#pragma unroll
      for (int j = 0; j < kElems; ++j) q[j] = 0.f;
#pragma unroll
    for (int j = 0; j < kElems; j += 4) s_vectors[(v * (kElems / 4) + j / 4) * threads + t] = make_float4(q[j], q[j + 1], q[j + 2], q[j + 3]);
  };
  // two pairs of a vector
  auto get = [&](int v, int j) { return *reinterpret_cast<const ulonglong2*>(s_vectors + (v * (kElems / 4) + j / 2) * threads + t); };
  if (team == 0) {
    put_vector(kWeight, a.weight, a.param_fp32);
    if (!RMS) put_vector(kBias, a.bias, a.param_fp32);
    if (POST) put_vector(kPostWeight, a.post_weight, a.param_fp32);
    if (POST && !RMS) put_vector(kPostBias, a.post_bias, a.param_fp32);
    if (channel_gate) put_vector(kGateVector, a.gate, a.gate_fp32);
  }
  if constexpr (!ONE)
    for (int i = threadIdx.x; i < int(sizeof(s_sums) / sizeof(float)); i += blockDim.x) s_sums[0][i] = 0.f;
  __syncthreads();

  // statistics of a row; afterwards v holds its normalised form, weighted
  auto normalise = [&](uint64_t (&v)[kPairs], float& mean, float& inv, int weight, int bias) {
    uint64_t sum = both(0.f);
    float total[1];
    mean = 0.f;
    if constexpr (!RMS) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) sum = add_f32x2(sum, v[j]);
      total[0] = fold(sum);
      team_sum(total);
      mean = total[0] * inv_hidden;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = add_f32x2(v[j], cols.inside(j, -mean));
      sum = both(0.f);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) sum = fma_f32x2(v[j], v[j], sum);
    total[0] = fold(sum);
    team_sum(total);
    inv = 1.f / sqrtf(fmaf(total[0], inv_hidden, a.eps));
    const uint64_t inv2 = both(inv);
#pragma unroll
    for (int j = 0; j < kPairs; j += 2) {
      const ulonglong2 w = get(weight, j);
      v[j] = mul_f32x2(v[j], inv2);
      v[j + 1] = mul_f32x2(v[j + 1], inv2);
      if constexpr (RMS) {
        v[j] = mul_f32x2(v[j], w.x);
        v[j + 1] = mul_f32x2(v[j + 1], w.y);
      } else {
        const ulonglong2 b = get(bias, j);
        v[j] = fma_f32x2(v[j], w.x, b.x);
        v[j + 1] = fma_f32x2(v[j + 1], w.y, b.y);
      }
    }
  };

#pragma unroll 1
  for (; row < a.rows; row += step) {
    const int64_t at = row * a.hidden;
    if constexpr (kRing) {
      ptx::copy_async_wait<kNormFwdRows - 1>();
#pragma unroll
      for (int i = 0; i < V; ++i) {
        reinterpret_cast<uint4*>(rx.w)[i] = s_ring[(slot * 2 * V + i) * 128];
        reinterpret_cast<uint4*>(rr.w)[i] = s_ring[(slot * 2 * V + V + i) * 128];
      }
      send(row + kNormFwdRows * step, slot);
      slot = slot + 1 == kNormFwdRows ? 0 : slot + 1;
    } else if constexpr (kAhead) {
      rx = nx;
      rr = nr;
      if (row + step < a.rows) fetch(row + step, nx, nr);
    } else {
      fetch(row, rx, rr);
    }
    uint64_t v[kPairs], p[kPairs];
    float4 stats = make_float4(0.f, 1.f, 0.f, 1.f);
    unpack(rx, v);
    if constexpr (POST) normalise(v, stats.x, stats.y, kPostWeight, kPostBias);
    if (channel_gate) {
#pragma unroll
      for (int j = 0; j < kPairs; j += 2) {
        const ulonglong2 g = get(kGateVector, j);
        v[j] = mul_f32x2(v[j], g.x);
        v[j + 1] = mul_f32x2(v[j + 1], g.y);
      }
    } else if (a.gate != nullptr) {
      cols.template load_param<T>(a.gate, a.gate_fp32, (int64_t)((uint32_t)row / a.gate_rows) * a.hidden, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = mul_f32x2(v[j], p[j]);
    }
    if (a.residual != nullptr) {
      const uint64_t scale = both(a.residual_scale);
      unpack(rr, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = fma_f32x2(scale, p[j], v[j]);
    }
    if (a.stream != nullptr) cols.store(static_cast<T*>(a.stream) + at, v);
    normalise(v, stats.z, stats.w, kWeight, kBias);
    cols.store(static_cast<T*>(a.normed) + at, v);
    if (a.stats != nullptr && t == 0) a.stats[row] = stats;
  }
}

template <typename T, bool RMS, bool POST, bool WIDE, int V, bool ONE>
int norm_fwd_launch_kernel(const ResidualNormArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> smem_done{0};
  auto kernel = residual_norm_kernel<T, RMS, POST, WIDE, V, ONE>;
  constexpr bool kRing = norm_fwd_ring<T>(RMS, POST, WIDE, V, ONE);
  constexpr int kRingBytes = kRing ? kNormFwdRows * 2 * V * 16 * 128 : 0, kMost = 5 * V * kRowElems * (ONE ? 32 : 256) * (int)sizeof(float) + kRingBytes;
  const int threads = a.teams * a.team_threads, smem = 5 * V * kRowElems * a.team_threads * (int)sizeof(float) + kRingBytes;
  const int64_t want = (a.rows + a.teams - 1) / a.teams, most = (int64_t)std::max(1, sm_count()) * (ONE ? norm_fwd_ctas(V, kRing) : 1);
  cudaError_t e = smem > 40 * 1024 ? allow_smem(smem_done, reinterpret_cast<const void*>(kernel), kMost) : cudaSuccess;
  if (e == cudaSuccess) e = launch_kernel<ResidualNormArgs>(kernel, a, dim3((unsigned)std::min(want, most)), threads, smem, false, s);
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "residual_norm launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

// Warps of a row, elements per thread and rows per CTA from the width.
template <typename T> int norm_fwd_launch(ResidualNormArgs a, bool wide, cudaStream_t s) {
  const int warps = (a.hidden + kNormFwdWarpElems - 1) / kNormFwdWarpElems;
  const int v = (a.hidden + warps * 32 * kRowElems - 1) / (warps * 32 * kRowElems);
  a.team_threads = warps * 32;
  a.teams = (warps == 1 ? 128 : kNormFwdThreads) / a.team_threads;
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
