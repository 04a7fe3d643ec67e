// Rows as 8-bit integers with a scale each (fdb_quantize_int8): scale = amax / 127, y = rint(x * (127 / amax)).
//
// A warp per row of up to 1024 elements, up to eight warps beyond (row_team.cuh); a row of up to 8192 is read once and stays in
// registers, a longer one is read a second time (it comes from L2 then).  HBM-bound: x read, one byte per element written.
// 16384 x 1024 bf16: 11.4 us = 4.4 TB/s.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "launch.h"
#include "quantize_int8.cuh"

namespace fdb {
namespace {

constexpr int kThreads = 128, kWarpElems = 1024;
constexpr int kMostCols = 1 << 30;  // columns are counted in 32 bits, up to a team's 8192 behind the last one

// Columns of an fp32 row that starts anywhere: runs of four per thread, so that what they become is stored four bytes at a time.
template <int V> struct QuadColumns {
  int t, threads, hidden;
  __device__ __forceinline__ int col(int j) const { return (t + j / 4 * threads) * 4 + j % 4; }
  __device__ __forceinline__ void load(const float* row, RowWords<float, V>& r) const {
#pragma unroll
    for (int j = 0; j < V * kRowElems; ++j) r.w[j] = col(j) < hidden ? __ldg(reinterpret_cast<const uint32_t*>(row) + col(j)) : 0u;
  }
};

struct QuantArgs {
  const void* x;
  uint8_t* y;
  float* scale;
  int64_t rows, pitch;
  int cols, team_threads, teams;
};

template <typename T, bool WIDE, int V>
__global__ void __launch_bounds__(256) quantize_int8_kernel(const __grid_constant__ QuantArgs a) {
  constexpr int kElems = V * kRowElems;
  constexpr bool kPieces = WIDE || sizeof(T) == 2;  // of eight elements
  using Columns = std::conditional_t<kPieces, RowColumns<row_mode<T>(WIDE), V>, QuadColumns<V>>;
  __shared__ uint32_t s_top[kThreads / 32][8];
  const int team = threadIdx.x / a.team_threads, t = threadIdx.x - team * a.team_threads;
  const int warps = a.team_threads / 32, span = a.team_threads * kElems;
  ptx::grid_launch();
  const int64_t row = (int64_t)blockIdx.x * a.teams + team;
  if (row < a.rows) {
    const T* x = static_cast<const T*>(a.x) + row * a.cols;
    uint32_t top = 0;
    RowWords<T, V> first;
    float v[kElems];
    for (int at = 0; at < a.cols; at += span) {
      const Columns cols{t, a.team_threads, a.cols - at};
      RowWords<T, V> r;
      cols.load(x + at, r);
      top = max(top, top_of(r));
      if (at == 0) first = r;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (warps > 1) {
      uint32_t* s = s_top[team];
      if ((threadIdx.x & 31) == 0) s[t >> 5] = top;
      ptx::bar_sync((uint32_t)team + 1, (uint32_t)a.team_threads);
      for (int w = 0; w < warps; ++w) top = max(top, s[w]);
    }
    const Int8Scale by = int8_scale<T>(top);
    if (t == 0) a.scale[row] = by.scale;
    for (int at = 0; at < a.cols; at += span) {
      const Columns cols{t, a.team_threads, a.cols - at};
      RowWords<T, V> r = first;
      if (at != 0) cols.load(x + at, r);
      unpack(r, v);
      if (!by.finite)
#pragma unroll
        for (int j = 0; j < kElems; ++j) v[j] = 0.f;  // (an infinity times zero is a NaN)
      uint8_t* y = a.y + row * a.pitch + at;
#pragma unroll
      for (int j = 0; j < kElems; j += kRowElems) {
        const uint2 o = make_uint2(four_bytes(v + j, by.inv), four_bytes(v + j + 4, by.inv));
        if constexpr (kPieces) {  // (up to seven zeros behind the row)
          if (cols.live(j)) *reinterpret_cast<uint2*>(y + cols.col(j)) = o;
        } else {
          if (cols.col(j) < cols.hidden) *reinterpret_cast<uint32_t*>(y + cols.col(j)) = o.x;
          if (cols.col(j + 4) < cols.hidden) *reinterpret_cast<uint32_t*>(y + cols.col(j + 4)) = o.y;
        }
      }
    }
  }
}

template <typename T, bool WIDE>
cudaError_t launch(const QuantArgs& a, int v, cudaStream_t s) {
  const int threads = a.teams * a.team_threads;
  const unsigned grid = (unsigned)((a.rows + a.teams - 1) / a.teams);
  if (v == 1) quantize_int8_kernel<T, WIDE, 1><<<grid, threads, 0, s>>>(a);
  else if (v == 2) quantize_int8_kernel<T, WIDE, 2><<<grid, threads, 0, s>>>(a);
  else if (v == 3) quantize_int8_kernel<T, WIDE, 3><<<grid, threads, 0, s>>>(a);
  else quantize_int8_kernel<T, WIDE, 4><<<grid, threads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

int launch_quantize_int8(const void* x, int dtype, int64_t rows, int cols, void* y, int64_t pitch, float* scale, void* stream) {
  QuantArgs a = {x, static_cast<uint8_t*>(y), scale, rows, pitch, cols, 0, 0};
  const int warps = std::min(8, (cols + kWarpElems - 1) / kWarpElems), v = std::min(4, (cols + warps * 256 - 1) / (warps * 256));
  a.team_threads = warps * 32;
  a.teams = std::max(1, kThreads / a.team_threads);
  const bool wide = cols % kRowElems == 0 && aligned_to(dtype == FDB_FP32 ? 32 : 16, x);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FDB_QUANT(T) (wide ? launch<T, true>(a, v, s) : launch<T, false>(a, v, s))
  const cudaError_t e = dtype == FDB_BF16 ? FDB_QUANT(__nv_bfloat16) : (dtype == FDB_FP16 ? FDB_QUANT(__half) : FDB_QUANT(float));
#undef FDB_QUANT
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "quantize_int8 launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

}  // namespace fdb

using namespace fdb;

extern "C" FDB_API int fdb_quantize_int8(const void* x, int32_t dtype, int64_t rows, int32_t cols, void* y, int64_t pitch, float* scale,
                                         void* stream) {
  clear_error();
  if (dtype != FDB_BF16 && dtype != FDB_FP16 && dtype != FDB_FP32) return fail(FDB_ERR_INVALID_ARGUMENT, "quantize_int8: dtype %d", dtype);
  if (rows > 2147483647LL || cols > kMostCols) return fail(FDB_ERR_LIMIT, "quantize_int8: %lld rows of %d; at most 2^31 - 1 of 2^30", (long long)rows, cols);
  if (rows < 0 || cols <= 0 || pitch < cols)
    return fail(FDB_ERR_INVALID_ARGUMENT, "quantize_int8: rows %lld, cols %d, pitch %lld", (long long)rows, cols, (long long)pitch);
  if (rows == 0) return FDB_OK;
  if (x == nullptr || y == nullptr || scale == nullptr) return fail(FDB_ERR_INVALID_ARGUMENT, "quantize_int8: x, y and scale must not be NULL");
  if (!aligned_to(dtype == FDB_FP32 ? 4 : 2, x) || !aligned_to(4, scale) || !aligned_to(16, y) || pitch % 16 != 0)
    return fail(FDB_ERR_ALIGNMENT, "quantize_int8: x and scale must be aligned to their elements, rows of y start on 16 bytes");
  return launch_quantize_int8(x, dtype, rows, cols, y, pitch, scale, stream);
}
