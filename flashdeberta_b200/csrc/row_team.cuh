// Rows of activations held by teams of warps: eight elements of a row per thread, or V times eight; sums over the team.
//
// Where rows are read in pieces of eight, thread t holds columns 8 (t + i threads) .. + 7, i < V; otherwise columns t + j threads, j < 8 V, so
// that the lanes of a warp still read neighbours.
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

// How rows are read and written: single elements (fp32 that starts anywhere), pieces of eight (WIDE: every row starts on a piece), pieces
// of eight 16-bit elements that start anywhere (SHIFTED: two aligned 16-byte pieces are loaded and moved into place; on the way
// out neighbouring lanes put aligned pieces together, and only the ends of a warp's run are written element by element).
enum : int { kRowSingle = 0, kRowWide = 1, kRowShifted = 2 };
template <typename T> constexpr int row_mode(bool wide) { return wide ? kRowWide : (sizeof(T) == 2 ? kRowShifted : kRowSingle); }

// Four words from byte `at` < 16 of eight.  (Selects, not branches: loads that come later can be issued before the words are there.)
__device__ __forceinline__ void shifted(const uint32_t (&c)[8], uint32_t at, uint32_t (&w)[4]) {
  uint32_t d[6], e[5];
#pragma unroll
  for (int k = 0; k < 6; ++k) d[k] = (at & 8u) != 0u ? c[k + 2] : c[k];
#pragma unroll
  for (int k = 0; k < 5; ++k) e[k] = (at & 4u) != 0u ? d[k + 1] : d[k];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(e[k], e[k + 1], (at & 3u) * 8u);
}

// Which columns of a row a thread holds.
template <int MODE, int V = 1> struct RowColumns {
  static constexpr int kElems = V * kRowElems;
  int t, threads, hidden;  // thread and threads of the team (whole warps)

  __device__ __forceinline__ int col(int j) const {
    if (MODE == kRowShifted) return (((t >> 5) * V + j / kRowElems) * 32 + (t & 31)) * kRowElems + j % kRowElems;
    return MODE == kRowWide ? (t + j / kRowElems * threads) * kRowElems + j % kRowElems : j * threads + t;
  }
  __device__ __forceinline__ bool live(int j) const { return col(MODE == kRowWide ? j / kRowElems * kRowElems : j) < hidden; }

  // The thread's elements of a row; zeros behind its end.
  template <typename T> __device__ __forceinline__ void load(const T* row, RowWords<T, V>& r) const {
    if constexpr (MODE == kRowWide) {
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
    } else if constexpr (MODE == kRowShifted) {
      const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;  // bytes; the same for every piece
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c0 = col(i * kRowElems), have = hidden - c0;
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + c0) - shift);
        // (an aligned piece with an element of the row in it never leaves the allocation)
        uint4 q = make_uint4(0, 0, 0, 0), n = q;
        if (have > 0) q = __ldg(p);
        if (2 * min(have, kRowElems) > 16 - (int)shift) n = __ldg(p + 1);
        const uint32_t c[8] = {q.x, q.y, q.z, q.w, n.x, n.y, n.z, n.w};
        uint32_t* w = r.w + i * 4;
        shifted(c, shift, *reinterpret_cast<uint32_t(*)[4]>(w));
        if (have < kRowElems)
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = 2 * k + 1 < have ? w[k] : (2 * k < have ? w[k] & 0xffffu : 0u);
      }
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int j = 0; j < kElems / 2; ++j) {
        const uint32_t lo = live(2 * j) ? __ldg(p + col(2 * j)) : 0u, hi = live(2 * j + 1) ? __ldg(p + col(2 * j + 1)) : 0u;
        r.w[j] = lo | (hi << 16);
      }
    }
  }
  // Bytes from <= b < to of an aligned piece (both even): whole words, and the half ones at the ends.
  static __device__ __forceinline__ void ends(char* p, const uint32_t (&o)[4], int from, int to) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * k >= from && 4 * k + 4 <= to) *reinterpret_cast<uint32_t*>(p + 4 * k) = o[k];
    auto word = [&](int k) { return k < 2 ? (k == 0 ? o[0] : o[1]) : (k == 2 ? o[2] : o[3]); };
    if ((from & 2) != 0) *reinterpret_cast<unsigned short*>(p + from) = (unsigned short)(word(from >> 2) >> 16);
    if ((to & 2) != 0 && to - 2 >= from) *reinterpret_cast<unsigned short*>(p + to - 2) = (unsigned short)word(to >> 2);
  }
  // (SHIFTED: by all lanes of a warp)
  template <typename T> __device__ __forceinline__ void store(T* row, const RowWords<T, V>& r) const {
    if constexpr (MODE == kRowWide) {
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
    } else if constexpr (MODE == kRowShifted) {
      // The warp's run: 32 V pieces from column c0 on, `bytes` of them in the row.  Aligned piece b begins 16 b - shift into the run, the end of
      // one lane's piece and the beginning of the next lane's; a lane keeps one that is not whole for the end (the first of the run and
      // the last of the row).
      const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
      const int lane = t & 31, c0 = (t >> 5) * V * 256, bytes = min(512 * V, 2 * (hidden - c0));
      char* run = reinterpret_cast<char*>(row + c0);
      uint32_t before[4] = {0u, 0u, 0u, 0u}, part[4] = {0u, 0u, 0u, 0u};  // lane 0: what lane 31 had; the piece that is kept
      int part_at = -16;
#pragma unroll
      for (int i = 0; i <= V; ++i) {
        uint32_t c[8], o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          c[k + 4] = i < V ? r.w[i < V ? i * 4 + k : 0] : 0u;
          const uint32_t left = i < V ? __shfl_sync(0xffffffffu, c[k + 4], (lane + 31) & 31) : 0u;
          c[k] = lane == 0 ? before[k] : left;
          before[k] = left;
        }
        shifted(c, 16u - shift, o);
        if (shift == 0u)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = c[k + 4];
        const int at = 16 * (32 * i + lane) - (int)shift;
        if (i == V && lane != 0) continue;
        if (at >= 0 && at + 16 <= bytes) {
          *reinterpret_cast<uint4*>(run + at) = make_uint4(o[0], o[1], o[2], o[3]);
        } else if (at < bytes && at + 16 > 0) {
          if (part_at > -16) ends(run + part_at, part, max(0, -part_at), min(16, bytes - part_at));  // (a lane that has both)
#pragma unroll
          for (int k = 0; k < 4; ++k) part[k] = o[k];
          part_at = at;
        }
      }
      if (part_at > -16) ends(run + part_at, part, max(0, -part_at), min(16, bytes - part_at));
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
    return MODE == kRowWide ? both(live(2 * pair) ? v : 0.f) : ptx::pack_f32x2(live(2 * pair) ? v : 0.f, live(2 * pair + 1) ? v : 0.f);
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
