// The 8-bit linear layer for a few tokens (fdb_linear_int8 with up to 32 rows, of integers up to 8): one launch, the rounding of the tokens
// included.
//
// What there is to do is to read the weight once and to wait for little else, so this kernel is built for latency: no tensor memory to
// allocate, no copies to set up, the weight goes straight into the registers of warp-level matrix instructions (mma.sync, 16 features
// x 8 tokens x 32), and its first loads are on their way before the tokens are looked at.  A CTA takes 16, 32 or 64 features, its
// eight warps share them and K; every CTA rounds all tokens to 8 bits itself, into shared memory (a few KB from L2, cheaper than a
// kernel in front).  The matrix instructions take K in any order as long as both operands take the same one: lane q of four holds 16
// consecutive bytes of each 64, so weight and tokens are read in 16-byte pieces.  The sums of the warps that share features are
// added up in shared memory, as integers, so their order changes nothing.  Measured: 1 x 768 -> 768 4.9 us, 1 x 1024 -> 4096 5.3,
// 8 x 1024 -> 4096 5.4, 1 x 4096 -> 4096 7.4 (an empty launch and its end take 2 to 3).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "gelu.cuh"
#include "internal.h"
#include "launch.h"
#include "linear_int8.h"
#include "quantize_int8.cuh"

namespace fdb {
namespace {

constexpr int kThreads = 256, kWarps = 8, kPrefetch = 4;  // chunks of 64 bytes of K whose weights a warp has on their way at first

struct SmallArgs {
  const void* x;
  int64_t x_pitch;       // bytes (int8) or elements between rows
  const float *x_scale, *w_scale;
  const uint8_t* weight;
  int64_t w_pitch;
  const void* bias;
  void* out;
  int rows, k, n, groups;  // groups: of 16 features a CTA takes, 1, 2 or 4
  int pitch;               // of the tokens in shared memory
  bool bias_fp32, wide, gelu;
};

__device__ __forceinline__ void mma_s8_16x8x32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Int8 {};  // the type of tokens that are integers already

// X: type of the tokens; TG: groups of eight of them
template <typename X, typename OUT, int TG>
__global__ void __launch_bounds__(kThreads) linear_int8_small_kernel(const __grid_constant__ SmallArgs a) {
  extern __shared__ __align__(16) uint8_t s_x[];  // 8 TG rows of `pitch` bytes; then the warps' sums
  __shared__ uint32_t s_top[kWarps];
  __shared__ float s_scale[8 * TG];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int splits = kWarps / a.groups, group = warp / splits, split = warp - group * splits;
  const int chunks = (a.k + 63) >> 6, c_first = chunks * split / splits, c_end = chunks * (split + 1) / splits;
  const int f0 = (blockIdx.x * a.groups + group) * 16;

  // the weight's rows g and g + 8 of the group (the last row where there is none: nobody stores what comes of it)
  const uint8_t* w0 = a.weight + (int64_t)min(f0 + g, a.n - 1) * a.w_pitch + 16 * q;
  const uint8_t* w1 = a.weight + (int64_t)min(f0 + g + 8, a.n - 1) * a.w_pitch + 16 * q;
  auto piece = [&](const uint8_t* w, int c) {
    return c < c_end && c * 64 + 16 * q < a.k ? __ldg(reinterpret_cast<const uint4*>(w + c * 64)) : make_uint4(0, 0, 0, 0);
  };
  uint4 ahead0[kPrefetch], ahead1[kPrefetch];
#pragma unroll
  for (int i = 0; i < kPrefetch; ++i) {
    ahead0[i] = piece(w0, c_first + i);
    ahead1[i] = piece(w1, c_first + i);
  }

  // the tokens as integers; zeros behind K and behind the last one
  const int padded = chunks * 64;
  if constexpr (sizeof(X) == 1) {
    for (int i = threadIdx.x; i < 8 * TG * (padded / 16); i += kThreads) {
      const int r = i / (padded / 16), at = (i - r * (padded / 16)) * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < a.rows && at < a.k) {
        v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.x) + r * a.x_pitch + at));
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int have = a.k - at - 4 * j;
          if (have < 4) w[j] &= have > 0 ? (1u << (8 * have)) - 1u : 0u;
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4*>(s_x + r * a.pitch + at) = v;
    }
    if (threadIdx.x < a.rows) s_scale[threadIdx.x] = __ldg(a.x_scale + threadIdx.x);
  } else {
    // As many warps per token as there are few tokens; 1024 elements of one at a time, the first of them kept in registers.
    constexpr int V = 4, kSpan = V * 256;
    const int at_once = a.rows > 4 ? 8 : (a.rows > 2 ? 4 : a.rows), share = kWarps / at_once, mine = warp % share;
    const int span = min(kSpan, (a.k + share * 256 - 1) / (share * 256) * 256);  // (a short token is spread over its warps)
    const int steps = (a.rows + at_once - 1) / at_once;
    for (int step = 0; step < steps; ++step) {
      const int r = step * at_once + warp / share;
      const bool has = r < a.rows;
      const X* x = static_cast<const X*>(a.x) + (int64_t)(has ? r : 0) * a.k;
      auto load = [&](int at, RowWords<X, V>& w) {
        const int left = max(0, min(span, a.k - at));
        if (a.wide) RowColumns<kRowWide, V>{lane, 32, left}.load(x + at, w);
        else RowColumns<kRowSingle, V>{lane, 32, left}.load(x + at, w);
      };
      RowWords<X, V> first, w;
      uint32_t top = 0;
      if (has) {
        load(mine * span, first);
        top = top_of(first);
        for (int at = (mine + share) * span; at < a.k; at += share * span) {
          load(at, w);
          top = max(top, top_of(w));
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (share > 1) {  // (every warp has the same number of steps)
        __syncthreads();
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
        for (int i = 0; i < share; ++i) top = max(top, s_top[warp / share * share + i]);
      }
      if (!has) continue;
      const Int8Scale by = int8_scale<X>(top);
      if (mine == 0 && lane == 0) s_scale[r] = by.scale;
      for (int at = mine * span; at < padded; at += share * span) {
        if (at == mine * span) w = first;
        else load(at, w);
        float v[V * kRowElems];
        unpack(w, v);
        if (!by.finite)
#pragma unroll
          for (int j = 0; j < V * kRowElems; ++j) v[j] = 0.f;
        uint8_t* s = s_x + r * a.pitch + at;
        const int room = min(span, padded - at);
#pragma unroll
        for (int j = 0; j < V * kRowElems; j += kRowElems) {
          const uint2 o = make_uint2(four_bytes(v + j, by.inv), four_bytes(v + j + 4, by.inv));
          if (a.wide) {
            const int c = RowColumns<kRowWide, V>{lane, 32, 0}.col(j);
            if (c < room) *reinterpret_cast<uint2*>(s + c) = o;
          } else {
#pragma unroll
            for (int i = 0; i < kRowElems; ++i) {
              const int c = RowColumns<kRowSingle, V>{lane, 32, 0}.col(j + i);
              if (c < room) s[c] = (uint8_t)((i < 4 ? o.x : o.y) >> (8 * (i % 4)));
            }
          }
        }
      }
    }
    // (rows behind the last token are multiplied and not stored: whatever they hold)
  }
  __syncthreads();

  int d[TG][4];
#pragma unroll
  for (int i = 0; i < TG; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0;
  for (int c = c_first; c < c_end; c += kPrefetch) {
#pragma unroll
    for (int i = 0; i < kPrefetch; ++i) {
      const uint4 u0 = ahead0[i], u1 = ahead1[i];
      ahead0[i] = piece(w0, c + i + kPrefetch);
      ahead1[i] = piece(w1, c + i + kPrefetch);
      if (c + i < c_end) {
#pragma unroll
        for (int t = 0; t < TG; ++t) {
          const uint4 b = *reinterpret_cast<const uint4*>(s_x + (8 * t + g) * a.pitch + (c + i) * 64 + 16 * q);
          mma_s8_16x8x32(d[t], u0.x, u1.x, u0.y, u1.y, b.x, b.y);
          mma_s8_16x8x32(d[t], u0.z, u1.z, u0.w, u1.w, b.z, b.w);
        }
      }
    }
  }

  // (group, split, feature, token)
  int* s_sum = reinterpret_cast<int*>(s_x + 8 * TG * a.pitch);
  {
    int* s = s_sum + warp * 16 * (8 * TG + 1);
#pragma unroll
    for (int t = 0; t < TG; ++t) {
      s[g * (8 * TG + 1) + 8 * t + 2 * q] = d[t][0];
      s[g * (8 * TG + 1) + 8 * t + 2 * q + 1] = d[t][1];
      s[(g + 8) * (8 * TG + 1) + 8 * t + 2 * q] = d[t][2];
      s[(g + 8) * (8 * TG + 1) + 8 * t + 2 * q + 1] = d[t][3];
    }
  }
  __syncthreads();
  const int features = a.groups * 16;
  for (int i = threadIdx.x; i < features * a.rows; i += kThreads) {
    const int f = i % features, r = i / features, n = blockIdx.x * features + f;
    if (n >= a.n) continue;
    const int* s = s_sum + (f / 16 * splits * 16 + f % 16) * (8 * TG + 1) + r;
    int sum = 0;
    for (int j = 0; j < splits; ++j) sum += s[j * 16 * (8 * TG + 1)];
    float b = 0.f;
    if (a.bias != nullptr) b = a.bias_fp32 ? __ldg(static_cast<const float*>(a.bias) + n) : to_float<OUT>(static_cast<const OUT*>(a.bias)[n]);
    float v = fmaf(__int2float_rn(sum) * __ldg(a.w_scale + n), s_scale[r], b), other;
    if (a.gelu) ptx::unpack_f32x2(sizeof(OUT) == 4 ? gelu_fine2(ptx::pack_f32x2(v, v)) : gelu_tail2(ptx::pack_f32x2(v, v)), v, other);
    static_cast<OUT*>(a.out)[(int64_t)r * a.n + n] = from_float<OUT>(v);
  }
}

template <typename X, typename OUT, int TG>
int launch(const SmallArgs& a, size_t smem, cudaStream_t s) {
  static std::atomic<uint64_t> smem_done{0};
  auto kernel = linear_int8_small_kernel<X, OUT, TG>;
  cudaError_t e = smem > 40 * 1024 ? allow_smem(smem_done, reinterpret_cast<const void*>(kernel), kInt8SmallSmem) : cudaSuccess;
  if (e == cudaSuccess) {
    const int features = 16 * a.groups;
    e = launch_kernel<SmallArgs>(kernel, a, dim3((unsigned)((a.n + features - 1) / features)), kThreads, smem, false, s);
  }
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "linear_int8 launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

template <typename X, typename OUT>
int launch_tokens(const SmallArgs& a, int tg, size_t smem, cudaStream_t s) {
  if constexpr (sizeof(X) == 1) return launch<X, OUT, 1>(a, smem, s);  // (int8_is_small: one round)
  else return tg == 1 ? launch<X, OUT, 1>(a, smem, s) : (tg == 2 ? launch<X, OUT, 2>(a, smem, s) : launch<X, OUT, 4>(a, smem, s));
}
template <typename X>
int launch_type(const SmallArgs& a, int out_dtype, int tg, size_t smem, cudaStream_t s) {
  if (out_dtype == FDB_BF16) return launch_tokens<X, __nv_bfloat16>(a, tg, smem, s);
  return out_dtype == FDB_FP16 ? launch_tokens<X, __half>(a, tg, smem, s) : launch_tokens<X, float>(a, tg, smem, s);
}

int token_groups(int64_t rows) { return rows <= 8 ? 1 : (rows <= 16 ? 2 : 4); }
// Rows 64 bytes past a multiple of 128: two tokens' pieces, read by eight lanes at once, lie on different banks.
int token_pitch(int k) { return (k + 63) / 64 % 2 == 0 ? (k + 63) / 64 * 64 + 64 : (k + 63) / 64 * 64; }
size_t small_smem(const fdb_linear_int8_params& p) {
  const int tg = token_groups(p.rows);
  return size_t(8 * tg) * token_pitch(p.in_features) + size_t(kWarps) * 16 * (8 * tg + 1) * sizeof(int);
}

}  // namespace

// Eight tokens are rounded at a time.  One such round always pays (8 x 4096 -> 1024: 9.0 us against 10.8 in two launches); several do as
// long as they stay short: 16 x 2048 -> 512 8.3 against 7.9, 29 x 768 -> 768 7.9 against 6.1 and 32 x 1024 -> 4096 9.5 against 6.7 on
// the device, where the second launch costs the host 5 us more; 16 x 4096 -> 1024 12.8 against 10.8.  Tokens that come as integers take
// one launch either way: 1 x 768 -> 768 4.2 against 4.7, 8 x 1024 -> 4096 5.3 against 5.6, 16 x 2048 -> 1024 7.5 against 6.5.
bool int8_is_small(const fdb_linear_int8_params& p) {
  if (p.rows > kInt8SmallRows || small_smem(p) > kInt8SmallSmem) return false;
  const int64_t rounds = (p.rows + 7) / 8;
  return rounds == 1 || (p.x_dtype != FDB_INT8 && rounds * p.in_features <= 4096);
}

int launch_linear_int8_small(const fdb_linear_int8_params& p, void* stream) {
  SmallArgs a;
  const bool given = p.x_dtype == FDB_INT8;
  const unsigned size = given ? 1 : (p.x_dtype == FDB_FP32 ? 4 : 2);
  a.x = p.x;
  a.x_pitch = p.x_pitch;
  a.x_scale = p.x_scale;
  a.w_scale = p.weight_scale;
  a.weight = static_cast<const uint8_t*>(p.weight);
  a.w_pitch = p.weight_pitch;
  a.bias = p.bias;
  a.out = p.out;
  a.rows = (int)p.rows;
  a.k = p.in_features;
  a.n = p.out_features;
  a.pitch = token_pitch(p.in_features);
  a.bias_fp32 = p.bias_dtype == FDB_FP32;
  a.wide = !given && p.in_features % kRowElems == 0 && aligned_to(8 * size, p.x);
  a.gelu = p.gelu != 0;
  const int groups = (p.out_features + 15) / 16, sms = std::max(1, sm_count());  // of all CTAs; two of them share an SM
  a.groups = groups <= 2 * sms ? 1 : (groups <= 4 * sms ? 2 : 4);
  const int tg = token_groups(p.rows);
  const size_t smem = small_smem(p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (given) return launch_type<Int8>(a, p.out_dtype, tg, smem, s);
  if (p.x_dtype == FDB_BF16) return launch_type<__nv_bfloat16>(a, p.out_dtype, tg, smem, s);
  return p.x_dtype == FDB_FP16 ? launch_type<__half>(a, p.out_dtype, tg, smem, s) : launch_type<float>(a, p.out_dtype, tg, smem, s);
}

}  // namespace fdb
