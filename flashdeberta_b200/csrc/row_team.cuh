// Rows of activations held by teams of warps: eight elements of a row per thread, sums over the team.
//
// A team is as many whole warps as a row of `hidden` elements needs at eight per thread.  Where rows may be read in 16-byte
// pieces (WIDE: hidden a multiple of 8, pointers 16-byte aligned) thread t holds columns 8t .. 8t+7; otherwise columns t,
// t + threads, t + 2 threads .., so that the lanes of a warp still read neighbouring elements.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace fdb {

constexpr int kRowElems = 8;         // elements of a row per thread
constexpr int kRowHiddenMax = 8192;  // 1024 threads

inline int row_team_threads(int hidden) { return (hidden + kRowElems * 32 - 1) / (kRowElems * 32) * 32; }

// Two elements in a 32-bit word (16-bit types) or one (fp32), as they lie in memory.
template <typename T> struct RowWords { uint32_t w[kRowElems * sizeof(T) / 4]; };

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void unpack(const RowWords<float>& r, float (&v)[kRowElems]) {
#pragma unroll
  for (int j = 0; j < kRowElems; ++j) v[j] = __uint_as_float(r.w[j]);
}
__device__ __forceinline__ void unpack(const RowWords<__nv_bfloat16>& r, float (&v)[kRowElems]) {
#pragma unroll
  for (int j = 0; j < kRowElems / 2; ++j) {
    v[2 * j] = __uint_as_float(r.w[j] << 16);
    v[2 * j + 1] = __uint_as_float(r.w[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const RowWords<__half>& r, float (&v)[kRowElems]) {
#pragma unroll
  for (int j = 0; j < kRowElems / 2; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void pack(const float (&v)[kRowElems], RowWords<float>& r) {
#pragma unroll
  for (int j = 0; j < kRowElems; ++j) r.w[j] = __float_as_uint(v[j]);
}
__device__ __forceinline__ void pack(const float (&v)[kRowElems], RowWords<__nv_bfloat16>& r) {
#pragma unroll
  for (int j = 0; j < kRowElems / 2; ++j) r.w[j] = ptx::pack_bf16x2(v[2 * j], v[2 * j + 1]);
}
__device__ __forceinline__ void pack(const float (&v)[kRowElems], RowWords<__half>& r) {
#pragma unroll
  for (int j = 0; j < kRowElems / 2; ++j) {
    const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    r.w[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Which columns of a row a thread holds.
template <bool WIDE> struct RowColumns {
  int t, threads, hidden;  // thread and threads of the team

  __device__ __forceinline__ int col(int j) const { return WIDE ? t * kRowElems + j : j * threads + t; }
  __device__ __forceinline__ bool live(int j) const { return WIDE ? t * kRowElems < hidden : j * threads + t < hidden; }

  // The thread's elements of a row; zeros behind its end.
  template <typename T> __device__ __forceinline__ void load(const T* row, RowWords<T>& r) const {
    constexpr int kWords = kRowElems * sizeof(T) / 4;
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (live(0)) q = __ldg(reinterpret_cast<const uint4*>(row + t * kRowElems) + i / 4);
        r.w[i] = q.x; r.w[i + 1] = q.y; r.w[i + 2] = q.z; r.w[i + 3] = q.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kRowElems; ++j) r.w[j] = live(j) ? __ldg(reinterpret_cast<const uint32_t*>(row) + col(j)) : 0u;
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const uint32_t lo = live(2 * j) ? __ldg(p + col(2 * j)) : 0u, hi = live(2 * j + 1) ? __ldg(p + col(2 * j + 1)) : 0u;
        r.w[j] = lo | (hi << 16);
      }
    }
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const RowWords<T>& r) const {
    constexpr int kWords = kRowElems * sizeof(T) / 4;
    if constexpr (WIDE) {
      if (!live(0)) return;
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        *(reinterpret_cast<uint4*>(row + t * kRowElems) + i / 4) = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kRowElems; ++j)
        if (live(j)) reinterpret_cast<uint32_t*>(row)[col(j)] = r.w[j];
    } else {
      unsigned short* p = reinterpret_cast<unsigned short*>(row);
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        if (live(2 * j)) p[col(2 * j)] = (unsigned short)(r.w[j] & 0xffffu);
        if (live(2 * j + 1)) p[col(2 * j + 1)] = (unsigned short)(r.w[j] >> 16);
      }
    }
  }
  template <typename T> __device__ __forceinline__ void load(const T* row, float (&v)[kRowElems]) const {
    RowWords<T> r;
    load(row, r);
    unpack(r, v);
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const float (&v)[kRowElems]) const {
    RowWords<T> r;
    pack(v, r);
    store(row, r);
  }
  // a vector over the columns, either of the rows' type or fp32
  template <typename T> __device__ __forceinline__ void load_param(const void* p, bool fp32, int64_t at, float (&v)[kRowElems]) const {
    if (fp32) load(static_cast<const float*>(p) + at, v);
    else load(static_cast<const T*>(p) + at, v);
  }
};

// Sums over the threads of a team, N values at a time.  `slots`: shared memory of the team, 2 x 32 x N floats: two halves in turn, so
// that one barrier a sum is enough (a half is written again only behind the barrier of the sum in between).
template <int N> struct TeamSum {
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
      for (int i = 0; i < N; ++i) s[i * 32 + warp] = v[i];
    ptx::bar_sync((uint32_t)barrier, (uint32_t)(warps * 32));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += s[i * 32 + w];
  }
};

}  // namespace fdb
