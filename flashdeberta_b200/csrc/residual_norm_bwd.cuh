// The row kernel of residual_norm's backward (the mathematics is at the head of residual_norm.cu), for one type of rows per
// translation unit.
#pragma once

#include "internal.h"
#include "launch.h"
#include "residual_norm.h"
#include "row_team.cuh"

namespace fdb {

using ptx::add_f32x2;
using ptx::fma_f32x2;
using ptx::mul_f32x2;

constexpr int kNormBwdTeams = kNormBwdThreads / 32;
constexpr size_t kNormBwdPlainSmem = 40 * 1024;  // with the 8 KB of the teams' sums, what a launch may take without being asked
constexpr int kNormBwdRows = 3;                  // of a team in shared memory: one that is worked on, two on their way

// Shared memory of a CTA: weight, post_weight, post_bias and a channel's gate in fp32 (read for every row, converted once), one vector of
// sums per thread for adding teams up and, where the gate has groups, what C = sum gate A and D = sum gate B have come to (touched
// only when a group ends).
__host__ __device__ constexpr size_t residual_norm_bwd_smem(int threads, int teams, bool post, int mode) {
  const size_t vector = size_t(threads) * kRowElems * sizeof(float), params = size_t(threads / teams) * kRowElems * sizeof(float);
  return 4 * params + (teams > 1 ? vector : 0) + (post && mode == kGateGroups ? 2 * vector : 0);
}

// Whether rows of 16-bit types are on their way in shared memory (the kernel says why), and what they take of it: x, residual, dnormed,
// dstream and an element's gate, 16 bytes of each per thread.  With what there is otherwise that is at most 200 KB.
__host__ __device__ constexpr bool norm_bwd_ring(bool post, int mode) { return post && mode != kGateChannel; }
__host__ __device__ constexpr size_t norm_bwd_ring_smem(int threads, int mode) { return size_t(kNormBwdRows) * (mode == kGateElement ? 5 : 4) * 16 * threads; }

template <typename T, bool RMS, bool POST, int GATE, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) residual_norm_bwd_kernel(const __grid_constant__ ResidualNormBwdArgs b) {
  constexpr int kPairs = kRowElems / 2;
  constexpr int kSums = RMS ? 1 : 2;  // per norm and row; and vectors of sums over rows: weight, bias
  extern __shared__ __align__(16) float s_vectors[];
  __shared__ __align__(16) float s_sums[kNormBwdTeams][TeamSum<kSums>::kSlots];
  const ResidualNormArgs& f = b.f;
  const int team = threadIdx.x / f.team_threads, t = threadIdx.x - team * f.team_threads;
  const RowColumns<row_mode<T>(WIDE)> cols{t, f.team_threads, f.hidden};
  TeamSum<kSums> team_sum{s_sums[team], f.team_threads / 32, t >> 5, team + 1, 0};
  const float inv_hidden = 1.f / (float)f.hidden;
  const int64_t worker = (int64_t)blockIdx.x * f.teams + team;
  const bool has_rows = worker < b.workers;
  const int64_t first = has_rows ? f.rows * worker / b.workers : 0, end = has_rows ? f.rows * (worker + 1) / b.workers : 0;
  ptx::grid_launch();

  // Rows on their way.  With a norm after the block and a gate per group or element there is much to keep in registers: rows come
  // through shared memory then, two ahead, by copies that nobody waits for until they are due; every thread copies what it reads
  // itself, so there is nothing to wait for but its own copies.  Otherwise the next row is on its way in registers while one is worked on.
  // 32768 x 1024 bf16, registers against shared memory, both LayerNorms: gate per group 114 and 101 us, per element 158 and 106, per
  // channel 96 and 110; one LayerNorm 81 and 84; RMS norms, gate per group 94 and 92.  fp32 rows and 1024 threads have room for neither
  // (8192 x 768 fp32: 40 us, through shared memory 49); single elements and shifted pieces are put into words at once.
  constexpr bool kPrefetch = sizeof(T) == 2 && WIDE && THREADS <= kNormBwdThreads;
  constexpr bool kRing = kPrefetch && norm_bwd_ring(POST, GATE), kAhead = kPrefetch && !kRing;
  constexpr int kTensors = GATE == kGateElement ? 5 : 4;
  enum : int { kX = 0, kResidual = 1, kDnormed = 2, kDstream = 3, kGateRow = 4 };
  const bool element_gate = GATE == kGateElement && f.gate != nullptr && !f.gate_fp32;
  uint4* s_ring = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(s_vectors) + b.ring_at) + threadIdx.x;
  auto slot_at = [&](int slot, int tensor) { return s_ring + (slot * kTensors + tensor) * blockDim.x; };
  auto copy = [&](const void* p, int64_t at, int slot, int tensor) {
    ptx::copy_async_16B(ptx::smem_u32(slot_at(slot, tensor)), static_cast<const T*>(p) + at + t * kRowElems);
  };
  auto send = [&](int64_t row, int slot) {
    if (row < end && cols.live(0)) {
      const int64_t at = row * f.hidden;
      copy(f.x, at, slot, kX);
      if (f.residual != nullptr) copy(f.residual, at, slot, kResidual);
      if (b.dnormed != nullptr) copy(b.dnormed, at, slot, kDnormed);
      if (b.dstream != nullptr) copy(b.dstream, at, slot, kDstream);
      if constexpr (GATE == kGateElement) { if (element_gate) copy(f.gate, at, slot, kGateRow); }
    }
    ptx::copy_async_commit();  // (a group per row, empty or not: they are counted)
  };
  struct Row { RowWords<T> tensor[kTensors]; float4 stats; };
  auto fetch = [&](int64_t row, Row& r) {
    const int64_t at = row * f.hidden;
    cols.load(static_cast<const T*>(f.x) + at, r.tensor[kX]);
    if (f.residual != nullptr) cols.load(static_cast<const T*>(f.residual) + at, r.tensor[kResidual]);
    if (b.dnormed != nullptr) cols.load(static_cast<const T*>(b.dnormed) + at, r.tensor[kDnormed]);
    if (b.dstream != nullptr) cols.load(static_cast<const T*>(b.dstream) + at, r.tensor[kDstream]);
    if constexpr (GATE == kGateElement) { if (element_gate) cols.load(static_cast<const T*>(f.gate) + at, r.tensor[kGateRow]); }
    r.stats = __ldg(f.stats + row);
  };
  int slot = 0;
  Row now, next;
  auto take = [&](int tensor, uint64_t (&v)[kPairs]) {
    if constexpr (kRing) {
      RowWords<T> r;
      *reinterpret_cast<uint4*>(r.w) = *slot_at(slot, tensor);
      unpack(r, v);
    } else {
      unpack(now.tensor[tensor], v);
    }
  };
  if constexpr (kRing) {
    if (!cols.live(0))  // a thread behind the end of the row reads zeros all the time
      for (int i = 0; i < kNormBwdRows * kTensors; ++i) s_ring[i * blockDim.x] = make_uint4(0, 0, 0, 0);
    for (int i = 0; i < kNormBwdRows - 1; ++i) send(first + i, i);
    if (first < end) now.stats = __ldg(f.stats + first);
  } else if constexpr (kAhead) {
    if (first < end) fetch(first, now);
  }

  // vectors over the columns: two 16-byte pieces per thread, each piece of the team's threads side by side
  enum : int { kWeight = 0, kPostWeight = 1, kPostBias = 2, kGateVector = 3 };
  auto vector_at = [&](int v) { return reinterpret_cast<float4*>(s_vectors) + v * 2 * f.team_threads + t; };
  auto put_vector = [&](int v, const void* p, bool fp32) {
    float q[kRowElems];
    if (p != nullptr) cols.template load_param<T>(p, fp32, 0, q);
    else
#pragma unroll
      for (int j = 0; j < kRowElems; ++j) q[j] = v == kGateVector ? 1.f : 0.f;
    vector_at(v)[0] = make_float4(q[0], q[1], q[2], q[3]);
    vector_at(v)[f.team_threads] = make_float4(q[4], q[5], q[6], q[7]);
  };
  auto get_vector = [&](int v, uint64_t (&q)[kPairs]) {
    const ulonglong2 lo = *reinterpret_cast<const ulonglong2*>(vector_at(v)), hi = *reinterpret_cast<const ulonglong2*>(vector_at(v) + f.team_threads);
    q[0] = lo.x; q[1] = lo.y; q[2] = hi.x; q[3] = hi.y;
  };
  if (team == 0) {
    put_vector(kWeight, f.weight, f.param_fp32);
    put_vector(kPostWeight, f.post_weight, f.param_fp32);
    put_vector(kPostBias, f.post_bias, f.param_fp32);
    put_vector(kGateVector, GATE == kGateChannel ? f.gate : nullptr, f.gate_fp32);
  }
  float* s_team = s_vectors + 4 * f.team_threads * kRowElems;
  float* s_C = s_team + (f.teams > 1 ? blockDim.x * kRowElems : 0) + threadIdx.x * kRowElems;
  float* s_D = s_C + blockDim.x * kRowElems;
  if constexpr (GATE == kGateGroups && POST) {
#pragma unroll
    for (int j = 0; j < kRowElems; ++j) s_C[j] = s_D[j] = 0.f;
  }
  for (int i = threadIdx.x; i < int(sizeof(s_sums) / sizeof(float)); i += blockDim.x) s_sums[0][i] = 0.f;
  __syncthreads();

  uint64_t sum_w[kPairs], sum_b[kPairs], sum_A[kPairs], sum_B[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) sum_w[j] = sum_b[j] = sum_A[j] = sum_B[j] = both(0.f);
  uint64_t* s_C2 = reinterpret_cast<uint64_t*>(s_C);
  uint64_t* s_D2 = reinterpret_cast<uint64_t*>(s_D);
  // A and B of a group leave the registers
  auto leave_group = [&](int64_t group, const uint64_t (&gate)[kPairs]) {
    float* slot = b.slots + (worker + group) * 2 * f.hidden;
    cols.store(slot, sum_A);
    if constexpr (!RMS) cols.store(slot + f.hidden, sum_B);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      if constexpr (POST) {
        s_C2[j] = fma_f32x2(gate[j], sum_A[j], s_C2[j]);
        if constexpr (!RMS) s_D2[j] = fma_f32x2(gate[j], sum_B[j], s_D2[j]);
      }
      sum_A[j] = sum_B[j] = both(0.f);
    }
  };

  int64_t group = -1;
  uint64_t g[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) g[j] = both(1.f);
  const uint64_t scale = both(f.residual_scale);
#pragma unroll(kAhead && RMS ? 2 : 1)  // (two rows a round save the copy of the words, 105 -> 95 us at 32768 x 1024; with a LayerNorm's sums they spill)
  for (int64_t row = first; row < end; ++row) {
    if constexpr (kRing) {
      send(row + kNormBwdRows - 1, slot == 0 ? kNormBwdRows - 1 : slot - 1);  // where the row before was
      if (row + 1 < end) next.stats = __ldg(f.stats + row + 1);
      ptx::copy_async_wait<kNormBwdRows - 1>();
    } else if constexpr (kAhead) {
      if (row + 1 < end) fetch(row + 1, next);
    } else {
      fetch(row, now);
    }
    const int64_t at = row * f.hidden;
    if constexpr (GATE == kGateGroups) {
      const int64_t mine = (uint32_t)row / f.gate_rows;
      if (mine != group) {
        if (group >= 0) leave_group(group, g);
        group = mine;
        cols.template load_param<T>(f.gate, f.gate_fp32, group * f.hidden, g);
      }
    } else if constexpr (GATE == kGateElement) {
      if (element_gate) take(kGateRow, g);
      else if (f.gate != nullptr) cols.load(static_cast<const float*>(f.gate) + at, g);
    } else {
      get_vector(kGateVector, g);
    }

    // the stream again; hat: x normalised (x itself without the norm), z: the stream normalised
    uint64_t hat[kPairs], u[kPairs], z[kPairs], d[kPairs], p[kPairs];
    take(kX, hat);
    if constexpr (POST) {
      const uint64_t mean = both(-now.stats.x), inv = both(now.stats.y);
      get_vector(kPostWeight, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        hat[j] = mul_f32x2(RMS ? hat[j] : add_f32x2(hat[j], mean), inv);
        u[j] = mul_f32x2(hat[j], p[j]);
      }
      if constexpr (!RMS) {
        get_vector(kPostBias, p);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) u[j] = add_f32x2(u[j], p[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) u[j] = hat[j];
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) z[j] = mul_f32x2(g[j], u[j]);
    if (f.residual != nullptr) {
      take(kResidual, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) z[j] = fma_f32x2(scale, p[j], z[j]);
    }
    {
      const uint64_t mean = both(-now.stats.z), inv = both(now.stats.w);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) z[j] = mul_f32x2(RMS ? z[j] : add_f32x2(z[j], mean), inv);
    }

    // dz, the gradient of the stream in all
    float sums[kSums];
    if (b.dnormed != nullptr) {
      uint64_t s0 = both(0.f), s1 = both(0.f);
      take(kDnormed, d);
      get_vector(kWeight, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        sum_w[j] = fma_f32x2(d[j], z[j], sum_w[j]);
        if constexpr (!RMS) sum_b[j] = add_f32x2(sum_b[j], d[j]);
        d[j] = mul_f32x2(d[j], p[j]);
        s0 = fma_f32x2(d[j], z[j], s0);
        if constexpr (!RMS) s1 = add_f32x2(s1, d[j]);
      }
      sums[kSums - 1] = fold(s1);
      sums[0] = fold(s0);
      team_sum(sums);
      // inv (y - mean(y) - z mean(y z)), the means scaled first
      const float scaled = now.stats.w * inv_hidden;
      const uint64_t inv = both(now.stats.w), m0 = both(-scaled * sums[0]), m1 = both(RMS ? 0.f : -scaled * sums[kSums - 1]);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[j] = fma_f32x2(d[j], inv, RMS ? mul_f32x2(z[j], m0) : fma_f32x2(z[j], m0, m1));
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[j] = both(0.f);
    }
    if (b.dstream != nullptr) {
      take(kDstream, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[j] = add_f32x2(d[j], p[j]);
    }
    if (b.dresidual != nullptr) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) p[j] = mul_f32x2(scale, d[j]);
      cols.store(static_cast<T*>(b.dresidual) + at, p);
    }
    if constexpr (GATE == kGateElement) {
      if (b.dgate != nullptr) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) p[j] = mul_f32x2(d[j], u[j]);
        if (f.gate_fp32) cols.store(static_cast<float*>(b.dgate) + at, p);
        else cols.store(static_cast<T*>(b.dgate) + at, p);
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[j] = mul_f32x2(d[j], g[j]);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      sum_A[j] = fma_f32x2(d[j], hat[j], sum_A[j]);
      if constexpr (!RMS) sum_B[j] = add_f32x2(sum_B[j], d[j]);
    }
    if constexpr (GATE != kGateElement) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[j] = mul_f32x2(d[j], g[j]);
    }
    if constexpr (POST) {
      uint64_t s0 = both(0.f), s1 = both(0.f);
      get_vector(kPostWeight, p);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        d[j] = mul_f32x2(d[j], p[j]);
        s0 = fma_f32x2(d[j], hat[j], s0);
        if constexpr (!RMS) s1 = add_f32x2(s1, d[j]);
      }
      sums[kSums - 1] = fold(s1);
      sums[0] = fold(s0);
      team_sum(sums);
      const float scaled = now.stats.y * inv_hidden;
      const uint64_t inv = both(now.stats.y), m0 = both(-scaled * sums[0]), m1 = both(RMS ? 0.f : -scaled * sums[kSums - 1]);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[j] = fma_f32x2(d[j], inv, RMS ? mul_f32x2(hat[j], m0) : fma_f32x2(hat[j], m0, m1));
    }
    cols.store(static_cast<T*>(b.dx) + at, d);
    if constexpr (kRing) {
      slot = slot + 1 == kNormBwdRows ? 0 : slot + 1;
      now.stats = next.stats;
    } else if constexpr (kAhead) {
      now = next;
    }
  }
  if constexpr (GATE == kGateGroups) {
    if (group >= 0) leave_group(group, g);
    if constexpr (POST) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        sum_A[j] = s_C2[j];
        sum_B[j] = s_D2[j];
      }
    }
  }

  // the CTA's sums
  float* part = b.parts + (int64_t)blockIdx.x * b.vectors * f.hidden;
  auto write = [&](const uint64_t (&v)[kPairs], int vector) {
    if (f.teams == 1) {
      cols.store(part + (int64_t)vector * f.hidden, v);
      return;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPairs; ++j) reinterpret_cast<uint64_t*>(s_team)[threadIdx.x * kPairs + j] = v[j];
    __syncthreads();
    const int all = f.team_threads * kRowElems;
    for (int i = threadIdx.x; i < all; i += blockDim.x) {
      const int c = row_mode<T>(WIDE) != kRowSingle ? i : (i % kRowElems) * f.team_threads + i / kRowElems;
      float sum = 0.f;
      for (int k = 0; k < f.teams; ++k) sum += s_team[k * all + i];
      if (c < f.hidden) part[(int64_t)vector * f.hidden + c] = sum;
    }
  };
  write(sum_w, 0);
  if constexpr (!RMS) write(sum_b, 1);
  write(sum_A, kSums);
  if constexpr (!RMS) write(sum_B, kSums + 1);
}

template <typename T, bool RMS, bool POST, int GATE, bool WIDE, int THREADS>
int norm_bwd_launch_kernel(ResidualNormBwdArgs b, cudaStream_t s) {
  static std::atomic<uint64_t> smem_done{0};
  constexpr bool kRing = sizeof(T) == 2 && WIDE && THREADS <= kNormBwdThreads && norm_bwd_ring(POST, GATE);
  // what the widest row of this form takes: asked for once, since calls of other widths on other host threads launch the same kernel
  constexpr int kMost = int(residual_norm_bwd_smem(THREADS, 1, POST, GATE) + (kRing ? norm_bwd_ring_smem(THREADS, GATE) : 0));
  auto kernel = residual_norm_bwd_kernel<T, RMS, POST, GATE, WIDE, THREADS>;
  const int threads = b.f.teams * b.f.team_threads;
  size_t smem = residual_norm_bwd_smem(threads, b.f.teams, POST, GATE);
  b.ring_at = (int)smem;
  if (kRing) smem += norm_bwd_ring_smem(threads, GATE);
  cudaError_t e = smem > kNormBwdPlainSmem ? allow_smem(smem_done, reinterpret_cast<const void*>(kernel), kMost) : cudaSuccess;
  if (e == cudaSuccess) e = launch_kernel<ResidualNormBwdArgs>(kernel, b, dim3((unsigned)b.ctas), threads, smem, false, s);
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "residual_norm backward launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

// WIDE stores of fp32 sums need rows of them to start on 16 bytes: they do, hidden being a multiple of 8 there.
template <typename T> int norm_bwd_launch(const ResidualNormBwdArgs& b, bool wide, cudaStream_t s) {
  const bool narrow = b.f.teams * b.f.team_threads <= kNormBwdThreads;
#define FDB_BWD4(R, P, G, W) (narrow ? norm_bwd_launch_kernel<T, R, P, G, W, kNormBwdThreads>(b, s) : norm_bwd_launch_kernel<T, R, P, G, W, 1024>(b, s))
#define FDB_BWD3(R, P, G) (wide ? FDB_BWD4(R, P, G, true) : FDB_BWD4(R, P, G, false))
#define FDB_BWD2(R, P) (b.mode == kGateChannel ? FDB_BWD3(R, P, kGateChannel) : (b.mode == kGateGroups ? FDB_BWD3(R, P, kGateGroups) : FDB_BWD3(R, P, kGateElement)))
  const bool post = b.f.post_weight != nullptr;
  if (b.f.rms) return post ? FDB_BWD2(true, true) : FDB_BWD2(true, false);
  return post ? FDB_BWD2(false, true) : FDB_BWD2(false, false);
#undef FDB_BWD4
#undef FDB_BWD3
#undef FDB_BWD2
}

}  // namespace fdb
