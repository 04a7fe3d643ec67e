// Norm over many tensors taken as one vector, and the tensors scaled to a bound on it (fdb_clip_grads): two launches for every thousand
// tensors (the norm alone: one, and one more for all).
//
// norm_kernel: the tensors are cut into chunks of 16384 elements, a CTA takes one run of chunks; squares (or magnitudes) are summed in
// fp32 over the 32 elements that a thread has in registers, those sums in fp64.  A sum of 32 that has left fp32's comfortable range
// (it would overflow, or squares have vanished) is taken again from the same registers in fp64, so gradients of any size count;
// zeros take that way too and cost nothing that memory does not hide.  One fp64 value per CTA goes to the workspace.
// scale_kernel: every CTA adds the values up itself, in the same order (a few KB from L2 in place of a third launch or a counter that
// somebody has to reset), and scales the chunks that it read in the first kernel, last one first: those are still in L2.  Where
// the factor is one, tensors that are their own output are left alone.
// The table of tensors travels as a kernel parameter: nothing to copy to the device or to keep until the kernel has read it.
// HBM-bound: every element read once for the norm, and read and written once where it is scaled.  Measured on 435 M bf16 gradients of 394
// tensors: norm 143 us = 6.1 TB/s, scaled into fp32 440 us = 5.9 TB/s; 38 small tensors 8 us for both launches.  Tensors that do not
// start on eight elements are read and written one by one: 1.4 to 1.7 times as long.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "launch.h"
#include "row_team.cuh"

namespace fdb {
namespace {

constexpr int kThreads = 512, kVectors = 4, kChunk = kThreads * kRowElems * kVectors;
constexpr int kCtasPerSm = 2;
// Entries of a table: kernel parameters hold 4 KB, or 32 KB (most tables) at a little more cost per launch.
constexpr int kSmallTable = 120, kLargeTable = 1000;

struct Entry {
  const void* data;
  void* out;
  int64_t count;
  uint32_t first_chunk;
  uint8_t dtype, out_dtype, wide, same;  // wide: both addresses allow pieces of eight elements; same: the tensor is its own output
};
template <int N> struct Table {
  double* partial;       // one value per CTA of every table
  float* norm;
  double max_norm;
  int n, mode;           // mode: 1, 2, or 0 for the largest magnitude
  uint32_t chunks;
  int partials, at;      // values in all, and where this table's begin
  Entry e[N];
};

// ---- a thread's 32 elements of a chunk ----
template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, int64_t left, bool wide, RowWords<T> (&r)[kVectors]) {
  if (wide && left >= kChunk) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const T* q = p + (i * kThreads + threadIdx.x) * kRowElems;
      if constexpr (sizeof(T) == 4) ptx::ld_global_32B(q, r[i].w);
      else *reinterpret_cast<uint4*>(r[i].w) = *reinterpret_cast<const uint4*>(q);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int64_t at = (int64_t)i * kThreads * kRowElems;
    const RowColumns<kRowSingle> cols{(int)threadIdx.x, kThreads, (int)max((int64_t)0, min(left - at, (int64_t)kThreads * kRowElems))};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kRowElems; ++j) r[i].w[j] = cols.live(j) ? reinterpret_cast<const uint32_t*>(p + at)[cols.col(j)] : 0u;
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p + at);
#pragma unroll
      for (int j = 0; j < kRowElems / 2; ++j) {
        const uint32_t lo = cols.live(2 * j) ? h[cols.col(2 * j)] : 0u, hi = cols.live(2 * j + 1) ? h[cols.col(2 * j + 1)] : 0u;
        r[i].w[j] = lo | (hi << 16);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ void store_vector(T* p, int64_t left, bool wide, int i, const float (&v)[kRowElems]) {
  RowWords<T> r;
  pack(v, r);
  if (wide && left >= kChunk) {
    T* q = p + (i * kThreads + threadIdx.x) * kRowElems;
    if constexpr (sizeof(T) == 4) ptx::st_global_32B(q, r.w);
    else *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(r.w);
    return;
  }
  const int64_t at = (int64_t)i * kThreads * kRowElems;
  const RowColumns<kRowSingle> cols{(int)threadIdx.x, kThreads, (int)max((int64_t)0, min(left - at, (int64_t)kThreads * kRowElems))};
  cols.store(p + at, r);
}

template <typename T>
__device__ __forceinline__ void add_chunk(const T* p, int64_t left, bool wide, int mode, double& sum, uint32_t& top) {
  RowWords<T> r[kVectors];
  load_chunk(p, left, wide, r);
  float v[kRowElems];
  if (mode == 0) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      unpack(r[i], v);
#pragma unroll
      for (int j = 0; j < kRowElems; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);  // (a NaN is larger than everything)
    }
    return;
  }
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    unpack(r[i], v);
#pragma unroll
    for (int j = 0; j < kRowElems; ++j) s[j & 1] = mode == 2 ? fmaf(v[j], v[j], s[j & 1]) : s[j & 1] + fabsf(v[j]);
  }
  const float all = s[0] + s[1];
  if (all > 1e-26f && all < 1e37f) {
    sum += (double)all;
  } else {
    for (int i = 0; i < kVectors; ++i) {
      unpack(r[i], v);
#pragma unroll
      for (int j = 0; j < kRowElems; ++j) sum += mode == 2 ? (double)v[j] * (double)v[j] : (double)fabsf(v[j]);
    }
  }
}

// The CTA's run of chunks, entry by entry; `back`: last chunk first.
template <int N, typename F>
__device__ __forceinline__ void for_chunks(const Table<N>& t, bool back, F&& f) {
  const uint32_t first = (uint32_t)((uint64_t)t.chunks * blockIdx.x / gridDim.x), end = (uint32_t)((uint64_t)t.chunks * (blockIdx.x + 1) / gridDim.x);
  if (first >= end) return;
  int lo = 0, hi = t.n - 1;  // the entry of the chunk to begin with: the last that starts at or before it
  const uint32_t begin = back ? end - 1 : first;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= begin) lo = mid; else hi = mid - 1;
  }
  if (back) {
    for (uint32_t c = end; c-- > first;) {
      while (t.e[lo].first_chunk > c) --lo;
      f(t.e[lo], (int64_t)(c - t.e[lo].first_chunk) * kChunk);
    }
  } else {
    for (uint32_t c = first; c < end; ++c) {
      while (lo + 1 < t.n && t.e[lo + 1].first_chunk <= c) ++lo;
      f(t.e[lo], (int64_t)(c - t.e[lo].first_chunk) * kChunk);
    }
  }
}

// Sum (or, mode 0, largest) of a value per thread, in every thread.  Magnitudes: larger bits, larger value, NaN largest.
__device__ __forceinline__ double join(double a, double b, int mode) {
  if (mode != 0) return a + b;
  return __double_as_longlong(a) > __double_as_longlong(b) ? a : b;
}
__device__ __forceinline__ double join_block(double v, int mode) {
  __shared__ double s[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), mode);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = join(v, s[w], mode);
  return v;
}

template <int N>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) norm_kernel(const __grid_constant__ Table<N> t) {
  ptx::grid_launch();
  double sum = 0.0;
  uint32_t top = 0;
  for_chunks(t, false, [&](const Entry& e, int64_t at) {
    const int64_t left = e.count - at;
    if (e.dtype == FDB_BF16) add_chunk(static_cast<const __nv_bfloat16*>(e.data) + at, left, e.wide, t.mode, sum, top);
    else if (e.dtype == FDB_FP16) add_chunk(static_cast<const __half*>(e.data) + at, left, e.wide, t.mode, sum, top);
    else add_chunk(static_cast<const float*>(e.data) + at, left, e.wide, t.mode, sum, top);
  });
  const double all = join_block(t.mode == 0 ? (double)__uint_as_float(top) : sum, t.mode);
  if (threadIdx.x == 0) t.partial[t.at + blockIdx.x] = all;
}

// The norm from the CTAs' values: the same in every CTA that asks.
__device__ __forceinline__ double total_norm(const double* partial, int n, int mode) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = join(v, partial[i], mode);
  v = join_block(v, mode);
  return mode == 2 ? sqrt(v) : v;
}

__global__ void __launch_bounds__(kThreads) norm_only_kernel(const double* partial, int n, int mode, float* norm) {
  ptx::grid_wait();
  const double v = total_norm(partial, n, mode);
  if (threadIdx.x == 0) *norm = (float)v;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const Entry& e, int64_t at, float factor) {
  const int64_t left = e.count - at;
  RowWords<T> r[kVectors];
  load_chunk(static_cast<const T*>(e.data) + at, left, e.wide, r);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float v[kRowElems];
    unpack(r[i], v);
#pragma unroll
    for (int j = 0; j < kRowElems; ++j) v[j] *= factor;
    if (e.out_dtype == FDB_BF16) store_vector(static_cast<__nv_bfloat16*>(e.out) + at, left, e.wide, i, v);
    else if (e.out_dtype == FDB_FP16) store_vector(static_cast<__half*>(e.out) + at, left, e.wide, i, v);
    else store_vector(static_cast<float*>(e.out) + at, left, e.wide, i, v);
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) scale_kernel(const __grid_constant__ Table<N> t) {
  ptx::grid_wait();
  const double norm = total_norm(t.partial, t.partials, t.mode);
  const double f = t.max_norm / (norm + 1e-6);
  const float factor = f >= 1.0 ? 1.f : (float)f;  // (a NaN stays one)
  if (t.at == 0 && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = (float)norm;
  for_chunks(t, true, [&](const Entry& e, int64_t at) {
    if (e.same && factor == 1.f) return;
    if (e.dtype == FDB_BF16) scale_chunk<__nv_bfloat16>(e, at, factor);
    else if (e.dtype == FDB_FP16) scale_chunk<__half>(e, at, factor);
    else scale_chunk<float>(e, at, factor);
  });
}

bool float_type(int t) { return t == FDB_BF16 || t == FDB_FP16 || t == FDB_FP32; }
unsigned type_bytes(int t) { return t == FDB_FP32 ? 4u : 2u; }

int validate_clip(const fdb_clip_grads_params* p) {
  if (p == nullptr || p->struct_bytes != sizeof(fdb_clip_grads_params))
    return fail(FDB_ERR_INVALID_ARGUMENT, "fdb_clip_grads_params: NULL or struct_bytes %u != %zu", p ? p->struct_bytes : 0u, sizeof(fdb_clip_grads_params));
  if (p->n_tensors < 0 || (p->n_tensors > 0 && p->tensors == nullptr) || p->norm_type < 0 || p->norm_type > 2)
    return fail(FDB_ERR_INVALID_ARGUMENT, "clip_grads: %d tensors, norm type %d", p->n_tensors, p->norm_type);
  if (p->scale != 0 && !(p->max_norm >= 0.0)) return fail(FDB_ERR_INVALID_ARGUMENT, "clip_grads: max_norm must not be negative or NaN");
  for (int i = 0; i < p->n_tensors; ++i) {
    const fdb_grad_tensor& g = p->tensors[i];
    if (!float_type(g.dtype) || g.count < 0 || (g.count > 0 && g.data == nullptr) ||
        (p->scale != 0 && (!float_type(g.out_dtype) || (g.count > 0 && g.out == nullptr) || (g.out == g.data && g.count > 0 && g.out_dtype != g.dtype))))
      return fail(FDB_ERR_INVALID_ARGUMENT, "clip_grads: tensor %d has a bad pointer, size or type", i);
    if (!aligned_to(type_bytes(g.dtype), g.data) || (p->scale != 0 && !aligned_to(type_bytes(g.out_dtype), g.out)))
      return fail(FDB_ERR_ALIGNMENT, "clip_grads: tensor %d is not aligned to its elements", i);
    if (g.count > (int64_t(1) << 44)) return fail(FDB_ERR_LIMIT, "clip_grads: tensor %d has %lld elements", i, (long long)g.count);
  }
  return FDB_OK;
}

// CTAs per table: the same for every call on a device, so that the workspace's size does not depend on the tensors' sizes.
int table_ctas() { return std::max(1, sm_count()) * kCtasPerSm; }
int tables_of(int n) { return std::max(1, (n + kLargeTable - 1) / kLargeTable); }

// Fills a table with the tensors from `first` on; false: too many chunks for one table.
template <int N> bool fill(Table<N>* t, const fdb_clip_grads_params& p, int first, int n) {
  uint64_t chunks = 0;
  t->n = 0;
  for (int i = first; i < first + n; ++i) {
    const fdb_grad_tensor& g = p.tensors[i];
    if (g.count == 0) continue;
    Entry& e = t->e[t->n++];
    e.data = g.data;
    e.out = g.out;
    e.count = g.count;
    e.first_chunk = (uint32_t)chunks;
    e.dtype = (uint8_t)g.dtype;
    e.out_dtype = (uint8_t)g.out_dtype;
    e.wide = aligned_to(8 * type_bytes(g.dtype), g.data) && (p.scale == 0 || aligned_to(8 * type_bytes(g.out_dtype), g.out));
    e.same = g.out == g.data;
    chunks += (uint64_t)((g.count + kChunk - 1) / kChunk);
    if (chunks > 0xffffffffull) return false;
  }
  t->chunks = (uint32_t)chunks;
  return true;
}

template <int N>
int run(const fdb_clip_grads_params& p, cudaStream_t s) {
  const int tables = tables_of(p.n_tensors), most = table_ctas();
  Table<N> t;
  t.partial = static_cast<double*>(p.workspace);
  t.norm = p.norm;
  t.max_norm = p.max_norm;
  t.mode = p.norm_type;
  int grids = 0;
  cudaError_t e = cudaSuccess;
  auto each = [&](auto&& go) {
    for (int k = 0, at = 0; k < tables && e == cudaSuccess; ++k) {
      const int first = k * kLargeTable;
      if (!fill(&t, p, first, std::min(p.n_tensors - first, tables > 1 ? kLargeTable : p.n_tensors))) return false;
      const int grid = (int)std::max<uint32_t>(1u, std::min<uint32_t>(t.chunks, (uint32_t)most));
      t.at = at;
      e = go(grid);
      at += grid;
      grids = at;
    }
    return true;
  };
  if (!each([&](int grid) { return launch_kernel<Table<N>>(norm_kernel<N>, t, dim3((unsigned)grid), kThreads, 0, false, s); }))
    return fail(FDB_ERR_LIMIT, "clip_grads: too many elements");
  // the last launch may start early; with several tables it may not, its wait covers the launch in front of it alone
  t.partials = grids;
  if (e == cudaSuccess) {
    if (p.scale != 0) {
      each([&](int grid) { return launch_kernel<Table<N>>(scale_kernel<N>, t, dim3((unsigned)grid), kThreads, 0, tables == 1, s); });
    } else {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1);
      cfg.blockDim = dim3(kThreads);
      cfg.stream = s;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at;
      cfg.numAttrs = tables == 1 ? 1 : 0;
      e = cudaLaunchKernelEx(&cfg, norm_only_kernel, (const double*)t.partial, grids, t.mode, t.norm);
    }
  }
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "clip_grads launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

}  // namespace
}  // namespace fdb

using namespace fdb;

extern "C" FDB_API uint64_t fdb_clip_grads_workspace_bytes(const fdb_clip_grads_params* p) {
  clear_error();
  if (validate_clip(p) != FDB_OK) return 0;
  return uint64_t(tables_of(p->n_tensors)) * table_ctas() * sizeof(double);
}

extern "C" FDB_API int fdb_clip_grads(const fdb_clip_grads_params* p, void* stream) {
  clear_error();
  const int rc = validate_clip(p);
  if (rc != FDB_OK) return rc;
  if (p->norm == nullptr) return fail(FDB_ERR_INVALID_ARGUMENT, "clip_grads: norm must not be NULL");
  if (!aligned_to(4, p->norm)) return fail(FDB_ERR_ALIGNMENT, "clip_grads: norm must be aligned to its element");
  const uint64_t need = uint64_t(tables_of(p->n_tensors)) * table_ctas() * sizeof(double);
  if (p->workspace == nullptr || p->workspace_bytes < need || !aligned_to(16, p->workspace))
    return fail(FDB_ERR_WORKSPACE, "clip_grads: workspace of %llu bytes needed (16-byte aligned), %llu given", (unsigned long long)need,
                (unsigned long long)p->workspace_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p->n_tensors <= kSmallTable ? run<kSmallTable>(*p, s) : run<kLargeTable>(*p, s);
}
