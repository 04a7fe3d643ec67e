// Rows of activations held by teams of warps: eight elements of a row per thread, or V times eight; sums over the team.
//
// Where eight elements may be read in one piece (WIDE: hidden a multiple of 8, pointers aligned to eight elements) thread t holds columns
// 8 (t + i threads) .. + 7, i < V; otherwise columns t + j threads, j < 8 V, so that the lanes of a warp still read neighbours.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace fdb {

constexpr int kRowElems = 8;
constexpr int kRowHiddenMax = 8192;

inline int row_team_threads(int hidden) { return (hidden + kRowElems * 32 - 1) / (kRowElems * 32) * 32; }

// Elements as they lie in memory: two in a 32-bit word (16-bit types) or one (fp32).
template <typename T, int V = 1> struct alignas(16) RowWords { uint32_t w[V * kRowElems * sizeof(T) / 4]; };

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <int N> __device__ __forceinline__ void unpack(const RowWords<float, N / kRowElems>& r, float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = __uint_as_float(r.w[j]);
}
template <int N> __device__ __forceinline__ void unpack(const RowWords<__nv_bfloat16, N / kRowElems>& r, float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    v[2 * j] = __uint_as_float(r.w[j] << 16);
    v[2 * j + 1] = __uint_as_float(r.w[j] & 0xffff0000u);
  }
}
template <int N> __device__ __forceinline__ void unpack(const RowWords<__half, N / kRowElems>& r, float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
template <int N> __device__ __forceinline__ void pack(const float (&v)[N], RowWords<float, N / kRowElems>& r) {
#pragma unroll
  for (int j = 0; j < N; ++j) r.w[j] = __float_as_uint(v[j]);
}
template <int N> __device__ __forceinline__ void pack(const float (&v)[N], RowWords<__nv_bfloat16, N / kRowElems>& r) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) r.w[j] = ptx::pack_bf16x2(v[2 * j], v[2 * j + 1]);
}
template <int N> __device__ __forceinline__ void pack(const float (&v)[N], RowWords<__half, N / kRowElems>& r) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    r.w[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The same as pairs of fp32 in 64-bit registers, for the two-wide arithmetic: half the instructions of a kernel that has to issue some
// forty per element.
template <typename T, int V> __device__ __forceinline__ void unpack(const RowWords<T, V>& r, uint64_t (&v)[V * kRowElems / 2]) {
  float f[V * kRowElems];
  unpack(r, f);
#pragma unroll
  for (int j = 0; j < V * kRowElems / 2; ++j) v[j] = ptx::pack_f32x2(f[2 * j], f[2 * j + 1]);
}
template <typename T, int V> __device__ __forceinline__ void pack(const uint64_t (&v)[V * kRowElems / 2], RowWords<T, V>& r) {
  float f[V * kRowElems];
#pragma unroll
  for (int j = 0; j < V * kRowElems / 2; ++j) ptx::unpack_f32x2(v[j], f[2 * j], f[2 * j + 1]);
  pack(f, r);
}
__device__ __forceinline__ uint64_t both(float v) { return ptx::pack_f32x2(v, v); }
__device__ __forceinline__ float fold(uint64_t v) {  // the sum of a pair
  float lo, hi;
  ptx::unpack_f32x2(v, lo, hi);
  return lo + hi;
}

// Which columns of a row a thread holds.
template <bool WIDE, int V = 1> struct RowColumns {
  static constexpr int kElems = V * kRowElems;
  int t, threads, hidden;  // thread and threads of the team

  __device__ __forceinline__ int col(int j) const {
    return WIDE ? (t + j / kRowElems * threads) * kRowElems + j % kRowElems : j * threads + t;
  }
  __device__ __forceinline__ bool live(int j) const { return col(WIDE ? j / kRowElems * kRowElems : j) < hidden; }

  // The thread's elements of a row; zeros behind its end.
  template <typename T> __device__ __forceinline__ void load(const T* row, RowWords<T, V>& r) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const T* p = row + col(i * kRowElems);
        if constexpr (sizeof(T) == 4) {
          uint32_t* w = r.w + i * 8;
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = 0u;
          if (live(i * kRowElems)) ptx::ld_global_32B(p, w);
        } else {
          uint4 q = make_uint4(0, 0, 0, 0);
          if (live(i * kRowElems)) q = __ldg(reinterpret_cast<const uint4*>(p));
          uint32_t* w = r.w + i * 4;
          w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
        }
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kElems; ++j) r.w[j] = live(j) ? __ldg(reinterpret_cast<const uint32_t*>(row) + col(j)) : 0u;
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) {
        const uint32_t lo = live(2 * j) ? __ldg(p + col(2 * j)) : 0u, hi = live(2 * j + 1) ? __ldg(p + col(2 * j + 1)) : 0u;
        r.w[j] = lo | (hi << 16);
      }
    }
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const RowWords<T, V>& r) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!live(i * kRowElems)) continue;
        if constexpr (sizeof(T) == 4) ptx::st_global_32B(row + col(i * kRowElems), r.w + i * 8);
        else *reinterpret_cast<uint4*>(row + col(i * kRowElems)) = make_uint4(r.w[i * 4], r.w[i * 4 + 1], r.w[i * 4 + 2], r.w[i * 4 + 3]);
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kElems; ++j)
        if (live(j)) reinterpret_cast<uint32_t*>(row)[col(j)] = r.w[j];
    } else {
      unsigned short* p = reinterpret_cast<unsigned short*>(row);
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) {
        if (live(2 * j)) p[col(2 * j)] = (unsigned short)(r.w[j] & 0xffffu);
        if (live(2 * j + 1)) p[col(2 * j + 1)] = (unsigned short)(r.w[j] >> 16);
      }
    }
  }
  template <typename T> __device__ __forceinline__ void load(const T* row, float (&v)[kElems]) const {
    RowWords<T, V> r;
    load(row, r);
    unpack(r, v);
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const float (&v)[kElems]) const {
    RowWords<T, V> r;
    pack(v, r);
    store(row, r);
  }
  template <typename T> __device__ __forceinline__ void load(const T* row, uint64_t (&v)[kElems / 2]) const {
    RowWords<T, V> r;
    load(row, r);
    unpack(r, v);
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const uint64_t (&v)[kElems / 2]) const {
    RowWords<T, V> r;
    pack(v, r);
    store(row, r);
  }
  // a number where the row has columns, zero behind its end
  __device__ __forceinline__ uint64_t inside(int pair, float v) const {
    return WIDE ? both(live(2 * pair) ? v : 0.f) : ptx::pack_f32x2(live(2 * pair) ? v : 0.f, live(2 * pair + 1) ? v : 0.f);
  }
  // a vector over the columns, either of the rows' type or fp32
  template <typename T, typename F> __device__ __forceinline__ void load_param(const void* p, bool fp32, int64_t at, F& v) const {
    if (fp32) load(static_cast<const float*>(p) + at, v);
    else load(static_cast<const T*>(p) + at, v);
  }
};

// Sums over the threads of a team, N values at a time (N = 1 or 2).  `slots`: 2 x 32 N floats of shared memory per team, zero at first
// (the team's warps write theirs, sums run over whole 16-byte pieces): two halves in turn, so that one barrier a sum is enough - a
// half is written again only behind the barrier of the sum in between.
template <int N> struct TeamSum {
  static constexpr int kSlots = 2 * 32 * N;
  float* slots;
  int warps, warp, barrier, turn;

  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (warps == 1) return;
    float* s = slots + turn * 32 * N;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[warp * N + i] = v[i];
    ptx::bar_sync((uint32_t)barrier, (uint32_t)(warps * 32));
    float4 q = *reinterpret_cast<const float4*>(s);
    for (int w = 4; w < warps * N; w += 4) {
      const float4 p = *reinterpret_cast<const float4*>(s + w);
      q.x += p.x; q.y += p.y; q.z += p.z; q.w += p.w;
    }
    if constexpr (N == 1) {
      v[0] = (q.x + q.y) + (q.z + q.w);
    } else {
      v[0] = q.x + q.z;
      v[1] = q.y + q.w;
    }
  }
};

}  // namespace fdb
