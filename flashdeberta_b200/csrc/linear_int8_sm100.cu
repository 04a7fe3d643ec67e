// out = act(x_scale[m] * weight_scale[n] * sum_k x[m][k] weight[n][k] + bias[n]) in 8-bit integers for sm_100a: the linear layers of an
// encoder whose weights are held in 8 bits (fdb_linear_int8).
//
// tcgen05.mma kind::i8, exact 32-bit sums in tensor memory.  The structure is linear_sm100.cu's: persistent grid; a tile is 128 rows
// (CG = 1) or 256 rows (CG = 2, a pair of CTAs on two SMs) x BN output features, K in steps of 128 bytes through a ring of stages:
//   warp 0  TMA, the CTA's 128 x 128 bytes of x and its BN / CG rows of the weight; what lies behind the ends arrives as zeros
//   warp 1  (of the pair's even CTA) tcgen05.mma, four per stage; two accumulators in tensor memory
//   the other warps: epilogue, 32 rows and 128, 64 or 32 columns each: both scales, bias, activation in fp32, one rounding, a TMA
//           store.  Scales and biases of the next tile are fetched while one is worked on.
// Bound by the tensor cores at the power limit where K is long, by the epilogue where it is short (4800 clocks a 256 x 256 tile, with the
// GELU 8700, against 680 per 128 of K).  Measured: 16384 x 4096 -> 4096 167 us = 3.30 POP/s (twice the measured bf16 rate is 3.31);
// 16384 x 4096 -> 1024 49 us = 2.81; 16384 x 1024 -> 4096 54 us = 2.55, with the GELU 66 us = 2.09 (fp32 results 72 and 92 us); 16384 x 256 -> 4096 32 us,
// 134 MB written.  On the way (16384 x 1024 -> 4096 with GELU, the product alone): eight epilogue warps that store from registers 137 us;
// sixteen 90; TMA stores 84; scales a tile ahead 73; tensor memory handed over without a cluster-wide release 66.
// Every wait is bounded; on a timeout the CTA raises FDB_DEV_TIMEOUT in the status word, frees its tensor memory and returns.
// No TMA multicast.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "gelu.cuh"
#include "internal.h"
#include "launch.h"
#include "linear_int8.h"
#include "row_team.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.cuh"

namespace fdb {
namespace {

using namespace ptx;

constexpr int kBM = 128, kBK = 128;
constexpr int kTmaWarp = 0, kMmaWarp = 1, kEpiWarp0 = 2;

struct Int8Args {
  CUtensorMap tm_x, tm_w, tm_out;
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  int32_t* status;
  int64_t rows;
  int k, n, tiles_n;
  bool bias_fp32;  // else of the output's type
  bool wide;       // rows of the output start on 16 bytes, scales and bias too
};

constexpr int kStoreBytes = 64;  // of a row, in one TMA store

template <int CG, int BN, int COLS> struct Tile {
  static constexpr uint32_t kBytesA = kBM * kBK, kBytesW = BN / CG * kBK, kStageBytes = kBytesA + kBytesW;
  static constexpr int kStages = BN == 256 ? 5 : (CG == 2 ? 7 : (BN == 128 ? 5 : 6));
  // the epilogue: columns of a warp; what of them lies in shared memory: 32 rows of a store's bytes, scales and biases
  static constexpr int kCols = COLS, kEpiWarps = BN * 4 / kCols, kThreads = 32 * (kEpiWarp0 + kEpiWarps);
  static constexpr uint32_t kTurnBytes = 32 * kStoreBytes, kColBytes = 2 * kCols * 4;
  static constexpr uint32_t kSmemTurn = kStages * kStageBytes, kSmemCols = kSmemTurn + kEpiWarps * kTurnBytes, kSmemBars = kSmemCols + kEpiWarps * kColBytes;
  enum : uint32_t { kBarFull = 0, kBarEmpty = kStages, kBarAccFull = 2 * kStages, kBarAccEmpty = 2 * kStages + 2, kNumBars = 2 * kStages + 4 };
  static constexpr uint32_t kSmemBytes = kSmemBars + 8 * kNumBars + 16 + 1024;  // + tensor-memory slot, abort flag, alignment slack
  static constexpr uint32_t kTmemCols = 2 * BN;
};

template <typename T> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A pair of columns: the sums scaled, bias added, activation.
template <typename OUT, bool GELU> __device__ __forceinline__ uint64_t finish_pair(uint32_t a0, uint32_t a1, uint64_t w_scale, uint64_t x_scale, uint64_t bias) {
  const uint64_t v = fma_f32x2(mul_f32x2(pack_f32x2(__int2float_rn((int)a0), __int2float_rn((int)a1)), w_scale), x_scale, bias);
  if constexpr (!GELU) return v;
  else if constexpr (sizeof(OUT) == 4) return gelu_fine2(v);
  else return gelu_tail2(v);
}

template <typename T> __device__ __forceinline__ float bias_at(const Int8Args& a, int n) {
  if (a.bias == nullptr) return 0.f;
  return a.bias_fp32 ? __ldg(static_cast<const float*>(a.bias) + n) : to_float<T>(static_cast<const T*>(a.bias)[n]);
}

// N columns of 32 rows per warp, each thread its own row, into shared memory, from where a TMA store takes a row's 64 bytes (16 columns of
// fp32, 32 of the others) and leaves out what lies behind the ends.  (Stores from registers touch 32 lines each: 81 us against 66 at
// 16384 x 1024 -> 4096.)  Piece p (16 bytes) of row r lies at piece p ^ (r / 2 % 4), the swizzle of the map's 64-byte rows: no bank
// conflicts.  `cols`: the scales, and the biases COLS behind them, in shared memory; AT, of the accumulator, and `first`, of the store: where
// the columns begin.
template <typename T, bool GELU, int COLS, int N, int AT, int A>
__device__ __forceinline__ void convert_rows(const uint32_t (&acc)[A], uint64_t sx, const float* cols, uint32_t* stage, int first, int lane) {
  constexpr int kPiece = 16 / int(sizeof(T));
#pragma unroll
  for (int p = 0; p < N / kPiece; ++p) {
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < kPiece; e += 4) {
      const int c = p * kPiece + e;
      const float4 ws = *reinterpret_cast<const float4*>(cols + c), b = *reinterpret_cast<const float4*>(cols + COLS + c);
      float v0, v1, v2, v3;
      unpack_f32x2(finish_pair<T, GELU>(acc[AT + c], acc[AT + c + 1], pack_f32x2(ws.x, ws.y), sx, pack_f32x2(b.x, b.y)), v0, v1);
      unpack_f32x2(finish_pair<T, GELU>(acc[AT + c + 2], acc[AT + c + 3], pack_f32x2(ws.z, ws.w), sx, pack_f32x2(b.z, b.w)), v2, v3);
      if constexpr (sizeof(T) == 4) {
        o[0] = __float_as_uint(v0); o[1] = __float_as_uint(v1); o[2] = __float_as_uint(v2); o[3] = __float_as_uint(v3);
      } else {
        o[e >> 1] = pack_pair<T>(v0, v1);
        o[(e >> 1) + 1] = pack_pair<T>(v2, v3);
      }
    }
    const int piece = first * int(sizeof(T)) / 16 + p;
    *reinterpret_cast<uint4*>(stage + lane * 16 + 4 * (piece ^ ((lane >> 1) & 3))) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// The same where a row starts anywhere: 32 x 32 results, turned in shared memory and written a row at a time across the lanes.  (A
// thread writing its own row element by element would touch 32 sectors with every store.)  fp32 in two halves of 16 rows, column c
// of row r in word 32 r + (c ^ r); 16-bit types two columns to a word, pair w of row r in word 16 r + (w ^ (r / 2 % 16)): neither side of
// the turn has two lanes on one bank.
template <typename T, bool GELU, int COLS>
__device__ __forceinline__ void store_turned(const Int8Args& a, const uint32_t (&acc)[32], int64_t row0, int n0, uint64_t sx, const float* cols, uint32_t* turn, int lane) {
  float v[32];
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float4 ws = *reinterpret_cast<const float4*>(cols + c), b = *reinterpret_cast<const float4*>(cols + COLS + c);
    unpack_f32x2(finish_pair<T, GELU>(acc[c], acc[c + 1], pack_f32x2(ws.x, ws.y), sx, pack_f32x2(b.x, b.y)), v[c], v[c + 1]);
    unpack_f32x2(finish_pair<T, GELU>(acc[c + 2], acc[c + 3], pack_f32x2(ws.z, ws.w), sx, pack_f32x2(b.z, b.w)), v[c + 2], v[c + 3]);
  }
  const int n = n0 + lane, rows = (int)min((int64_t)32, a.rows - row0);
  T* out = static_cast<T*>(a.out) + row0 * a.n + n;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if ((lane >> 4) == half)
#pragma unroll
        for (int c = 0; c < 32; ++c) turn[(lane & 15) * 32 + (c ^ (lane & 15))] = __float_as_uint(v[c]);
      __syncwarp();
      if (n < a.n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (half * 16 + r < rows) out[(int64_t)(half * 16 + r) * a.n] = __uint_as_float(turn[r * 32 + (lane ^ r)]);
      __syncwarp();
    }
  } else {
#pragma unroll
    for (int w = 0; w < 16; ++w) turn[lane * 16 + (w ^ ((lane >> 1) & 15))] = pack_pair<T>(v[2 * w], v[2 * w + 1]);
    __syncwarp();
    if (n < a.n)
#pragma unroll 16
      for (int r = 0; r < 32; ++r)
        if (r < rows) reinterpret_cast<unsigned short*>(out)[(int64_t)r * a.n] = (unsigned short)(turn[r * 16 + ((lane >> 1) ^ ((r >> 1) & 15))] >> (16 * (lane & 1)));
    __syncwarp();
  }
}

template <int CG, int BN, int COLS, typename OUT, bool GELU>
__global__ void __launch_bounds__(Tile<CG, BN, COLS>::kThreads, 1) linear_int8_kernel(const __grid_constant__ Int8Args args) {
  using T = Tile<CG, BN, COLS>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem - smem_u32(smem_raw));
  const int tid = threadIdx.x, warp = (int)uniform(uint32_t(tid) >> 5), lane = tid & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;

  auto bar = [&](uint32_t i) -> uint32_t { return smem + T::kSmemBars + 8u * i; };
  const uint32_t tmem_slot = smem + T::kSmemBars + 8u * T::kNumBars;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem_gen + T::kSmemBars + 8u * T::kNumBars + 8u);

  if (tid == 0) {
    *abort_flag = 0u;
    for (uint32_t i = 0; i < T::kNumBars; ++i) mbar_init(bar(i), (i >= T::kBarAccEmpty) ? uint32_t(T::kEpiWarps * CG) : 1u);
    fence_barrier_init();
    tma_prefetch_desc(&args.tm_x);
    tma_prefetch_desc(&args.tm_w);
  }
  if (warp == kMmaWarp) {
    if constexpr (CG == 2) { tmem_alloc_pair(tmem_slot, T::kTmemCols); tmem_relinquish_pair(); }
    else { tmem_alloc(tmem_slot, T::kTmemCols); tmem_relinquish(); }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = uniform(*reinterpret_cast<volatile uint32_t*>(smem_gen + T::kSmemBars + 8u * T::kNumBars));

  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const int kblocks = (args.k + kBK - 1) / kBK;
  const int num_tiles = (int)((args.rows + kBM * CG - 1) / (kBM * CG)) * args.tiles_n;
  auto load_w = [&](uint32_t st, int kb, int n0) {
    const uint32_t w = smem + st * T::kStageBytes + T::kBytesA;
    if constexpr (CG == 2) {
      if (rank == 0) mbar_expect_tx(bar(T::kBarFull + st), 2 * T::kStageBytes);
      tma_load_2d_pair(w, &args.tm_w, bar(T::kBarFull + st), kb * kBK, n0);
    } else {
      mbar_expect_tx(bar(T::kBarFull + st), T::kStageBytes);
      tma_load_2d(w, &args.tm_w, bar(T::kBarFull + st), kb * kBK, n0);
    }
  };
  // The weight is nobody's output: its first stages are on their way before the kernel in front, which rounds x, has finished.
  const int early = kblocks < T::kStages ? kblocks : T::kStages;
  if (warp == kTmaWarp) {
    const int n0 = (first % args.tiles_n) * BN + int(rank) * (BN / CG);
#pragma unroll 1
    for (int kb = 0; kb < early; ++kb)
      if (elect_one()) load_w(uint32_t(kb), kb, n0);
  }
  grid_wait();
  bool ok = true;
  auto wait = [&](uint32_t b, uint32_t parity) {
    if (ok) ok = mbar_wait_warp(b, parity, abort_flag);
  };

  if (warp == kTmaWarp) {
    uint32_t st = 0, phase = 0;
    int skip = early;  // stages whose weights are already on their way
#pragma unroll 1
    for (int tile = first; tile < num_tiles && ok; tile += step) {
      const int m0 = (tile / args.tiles_n) * (kBM * CG) + int(rank) * kBM;
      const int n0 = (tile % args.tiles_n) * BN + int(rank) * (BN / CG);
#pragma unroll 1
      for (int kb = 0; kb < kblocks; ++kb) {
        if (skip == 0) wait(bar(T::kBarEmpty + st), phase ^ 1u);  // (the first round passes at once)
        if (!ok) break;
        if (elect_one()) {
          if (skip == 0) load_w(st, kb, n0);
          if constexpr (CG == 2) tma_load_2d_pair(smem + st * T::kStageBytes, &args.tm_x, bar(T::kBarFull + st), kb * kBK, m0);
          else tma_load_2d(smem + st * T::kStageBytes, &args.tm_x, bar(T::kBarFull + st), kb * kBK, m0);
        }
        skip -= skip > 0 ? 1 : 0;
        if (++st == T::kStages) { st = 0; phase ^= 1u; }
      }
    }
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint32_t idesc = instr_desc_s8(kBM * CG, BN);
      const uint64_t da0 = smem_desc_sw128(smem, 1024, 16), dw0 = smem_desc_sw128(smem + T::kBytesA, 1024, 16);
      uint32_t st = 0, phase = 0, local = 0;
#pragma unroll 1
      for (int tile = first; tile < num_tiles && ok; tile += step, ++local) {
        const uint32_t acc = local & 1u, d = tmem_base + acc * BN;
        wait(bar(T::kBarAccEmpty + acc), ((local >> 1) & 1u) ^ 1u);  // the epilogue has read this accumulator
        tc_fence_after();
#pragma unroll 1
        for (int kb = 0; kb < kblocks; ++kb) {
          wait(bar(T::kBarFull + st), phase);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = da0 + uint64_t(st * (T::kStageBytes >> 4)), dw = dw0 + uint64_t(st * (T::kStageBytes >> 4));
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              const uint32_t more = (kb > 0 || ks > 0) ? 1u : 0u;
              if constexpr (CG == 2) mma_s8_pair(d, da + uint64_t((ks * 32) >> 4), dw + uint64_t((ks * 32) >> 4), idesc, more);
              else mma_s8(d, da + uint64_t((ks * 32) >> 4), dw + uint64_t((ks * 32) >> 4), idesc, more);
            }
            if constexpr (CG == 2) mma_commit_pair(bar(T::kBarEmpty + st)); else mma_commit(bar(T::kBarEmpty + st));
            if (kb == kblocks - 1) { if constexpr (CG == 2) mma_commit_pair(bar(T::kBarAccFull + acc)); else mma_commit(bar(T::kBarAccFull + acc)); }
          }
          if (++st == T::kStages) { st = 0; phase ^= 1u; }
        }
      }
    }
  } else {
    const int quarter = warp & 3;                // the 32 tensor-memory lanes this warp may read
    const int mine = warp - kEpiWarp0, part = mine >> 2;
    constexpr int kCols = T::kCols, kStore = kStoreBytes / int(sizeof(OUT));  // this warp's columns of the tile; those of a store
    const uint32_t tmem_lane = tmem_base + (uint32_t(quarter * 32) << 16);
    uint32_t* turn = reinterpret_cast<uint32_t*>(smem_gen + T::kSmemTurn + mine * T::kTurnBytes);
    float* cols = reinterpret_cast<float*>(smem_gen + T::kSmemCols + mine * T::kColBytes);
    uint32_t acc_empty[2] = {bar(T::kBarAccEmpty), bar(T::kBarAccEmpty + 1)};
    if constexpr (CG == 2) { acc_empty[0] = map_to_rank(acc_empty[0], 0); acc_empty[1] = map_to_rank(acc_empty[1], 0); }
    uint32_t local = 0;
    // scales and biases of a tile's columns, a column (or two) per lane: fetched a tile ahead, put into shared memory when their turn comes
    float ws[kCols / 32], b[kCols / 32], x_scale = 0.f;
    auto fetch = [&](int tile) {
      const int64_t row = (int64_t)(tile / args.tiles_n) * (kBM * CG) + int(rank) * kBM + quarter * 32 + lane;
      const int n0 = (tile % args.tiles_n) * BN + part * kCols + lane;
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const bool has = tile < num_tiles && n0 + i * 32 < args.n;
        ws[i] = has ? __ldg(args.w_scale + n0 + i * 32) : 0.f;
        b[i] = has ? bias_at<OUT>(args, n0 + i * 32) : 0.f;
      }
      x_scale = tile < num_tiles && row < args.rows ? __ldg(args.x_scale + row) : 0.f;
    };
    fetch(first);
#pragma unroll 1
    for (int tile = first; tile < num_tiles; tile += step, ++local) {
      const int64_t row0 = (int64_t)(tile / args.tiles_n) * (kBM * CG) + int(rank) * kBM + quarter * 32;
      const int n0 = (tile % args.tiles_n) * BN + part * kCols;
      const uint32_t acc = local & 1u;
      const uint64_t sx = pack_f32x2(x_scale, x_scale);
      __syncwarp();  // (the tile before has been read from here)
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        cols[i * 32 + lane] = ws[i];
        cols[kCols + i * 32 + lane] = b[i];
      }
      __syncwarp();
      fetch(tile + step);
      wait(bar(T::kBarAccFull + acc), (local >> 1) & 1u);
      tc_fence_after();
      const bool has_rows = ok && row0 < args.rows;
      const uint32_t acc_at = tmem_lane + acc * BN + uint32_t(part * kCols);
      auto release = [&] {  // the accumulator is in registers: the next tile but one may overwrite it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) { if constexpr (CG == 2) mbar_arrive_peer(acc_empty[acc]); else mbar_arrive(acc_empty[acc]); }
      };
      auto begin_store = [&] {  // the store before has left the stage (the lane that issues them waits)
        tma_store_wait_read();
        __syncwarp();
      };
      auto end_store = [&](int at) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && n0 + at < args.n) {
          tma_store_2d(&args.tm_out, smem_u32(turn), n0 + at, (int)row0);
          tma_store_commit();
        }
      };
      if (kCols == 128 && args.wide) {  // few warps with many registers: the next 16 columns leave tensor memory while 16 are worked on
        uint32_t a0[16], a1[16];
        auto load = [&](int at, uint32_t (&a)[16]) { if (ok) tmem_ld16(acc_at + uint32_t(at), a); };
        load(0, a0);
        tmem_wait_ld();
#pragma unroll 1
        for (int at = 0; at < kCols; at += 32) {
          const bool live = has_rows && n0 + at < args.n;
          load(at + 16, a1);
          if (live) {
            begin_store();
            convert_rows<OUT, GELU, kCols, 16, 0>(a0, sx, cols + at, turn, 0, lane);
            if constexpr (kStore == 16) {
              end_store(at);
              begin_store();
            }
          }
          tmem_wait_ld();
          if (at + 32 < kCols) load(at + 32, a0); else release();
          if (live) {
            convert_rows<OUT, GELU, kCols, 16, 0>(a1, sx, cols + at + 16, turn, 16 % kStore, lane);
            end_store(at + 32 - kStore);
          }
          tmem_wait_ld();
        }
      } else {
#pragma unroll 1
        for (int at = 0; at < kCols; at += 32) {
          uint32_t a[32];
          if (ok) {  // whole warps execute the load, whatever their rows
            tmem_ld32(acc_at + uint32_t(at), a);
            tmem_wait_ld();
          }
          if (at + 32 == kCols) release();
          if (!has_rows || n0 + at >= args.n) continue;
          if (!args.wide) {
            store_turned<OUT, GELU, kCols>(args, a, row0, n0 + at, sx, cols + at, turn, lane);
            continue;
          }
          if constexpr (kCols == 128) continue;  // (done above)
          begin_store();
          convert_rows<OUT, GELU, kCols, kStore, 0>(a, sx, cols + at, turn, 0, lane);
          end_store(at);
          if constexpr (kStore == 16) {
            begin_store();
            convert_rows<OUT, GELU, kCols, kStore, 16>(a, sx, cols + at + 16, turn, 0, lane);
            end_store(at + 16);
          }
        }
      }
    }
  }
  if (warp >= kEpiWarp0 && lane == 0) tma_store_wait();

  // ---- teardown ----
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0u) {
    if (tid == 0 && args.status != nullptr) atomicOr(reinterpret_cast<unsigned int*>(args.status), FDB_DEV_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies and MMAs in flight get a bounded time to land
    __syncthreads();
  }
  if constexpr (CG == 2) {
    cluster_sync();  // the pair's arrivals on this CTA's barriers have landed, and both are done with tensor memory
    if (warp == kMmaWarp) tmem_dealloc_pair(tmem_base, T::kTmemCols);
  } else {
    if (warp == kMmaWarp) tmem_dealloc(tmem_base, T::kTmemCols);
  }
}

template <int CG, int BN, int COLS, typename OUT, bool GELU>
int launch(const Int8Args& a, int grid, bool chained, cudaStream_t stream) {
  using T = Tile<CG, BN, COLS>;
  static std::atomic<uint64_t> smem_done{0};
  auto kernel = linear_int8_kernel<CG, BN, COLS, OUT, GELU>;
  cudaError_t e = allow_smem(smem_done, reinterpret_cast<const void*>(kernel), (int)T::kSmemBytes);
  if (e == cudaSuccess) e = launch_kernel<Int8Args>(kernel, a, dim3((unsigned)grid), T::kThreads, T::kSmemBytes, chained, stream, CG);
  if (e != cudaSuccess) return fail(FDB_ERR_CUDA, "linear_int8 launch: %s", cudaGetErrorString(e));
  return FDB_OK;
}

template <int CG, int BN, int COLS>
int launch_type(const Int8Args& a, int grid, int out_dtype, bool gelu, bool chained, cudaStream_t s) {
#define FDB_INT8_OUT(OUT) (gelu ? launch<CG, BN, COLS, OUT, true>(a, grid, chained, s) : launch<CG, BN, COLS, OUT, false>(a, grid, chained, s))
  if (out_dtype == FDB_BF16) return FDB_INT8_OUT(__nv_bfloat16);
  return out_dtype == FDB_FP16 ? FDB_INT8_OUT(__half) : FDB_INT8_OUT(float);
#undef FDB_INT8_OUT
}

// Tile shapes: clocks per 128 of K and clocks of a tile's epilogue (with the GELU 1.8 times those), as measured over whole waves
// (16384 x 4096 -> 4096: 169, 166, 194, 259, 391 us; 16384 x 256 -> 4096: 32, 38, 41, 40, 54).  One runs beside the other but for the
// first tile's main loop and the last one's epilogue.  The 256 x 256 tile has two forms of the epilogue: 16 warps of 64 columns hide more
// latency, 8 of 128 columns leave the main loop more of the issue slots.  16384 rows, 16 against 8 warps: 256 -> 4096 32 and 38 us,
// 1024 -> 4096 57 and 54, with the GELU 66 and 73, 2048 -> 4096 with the GELU 97 and 95.
struct Config { int cg, bn, cols, clocks, epilogue; };
constexpr Config kConfigs[] = {{2, 256, 64, 680, 4800}, {2, 256, 128, 640, 5300}, {2, 128, 32, 430, 2700}, {1, 128, 32, 535, 2650}, {1, 64, 32, 403, 1800}};

bool float_type(int t) { return t == FDB_BF16 || t == FDB_FP16 || t == FDB_FP32; }
unsigned type_bytes(int t) { return t == FDB_FP32 ? 4u : 2u; }
int64_t pitch_of(const fdb_linear_int8_params& p) { return (int64_t(p.in_features) + 127) / 128 * 128; }  // whole lines of memory
uint64_t rows_bytes(const fdb_linear_int8_params& p) { return (uint64_t(p.rows) * pitch_of(p) + 255) / 256 * 256; }

int validate_int8(const fdb_linear_int8_params* p) {
  if (p == nullptr || p->struct_bytes != sizeof(fdb_linear_int8_params))
    return fail(FDB_ERR_INVALID_ARGUMENT, "fdb_linear_int8_params: NULL or struct_bytes %u != %zu", p ? p->struct_bytes : 0u, sizeof(fdb_linear_int8_params));
  if ((p->x_dtype != FDB_INT8 && !float_type(p->x_dtype)) || !float_type(p->out_dtype) || (p->bias != nullptr && !float_type(p->bias_dtype)))
    return fail(FDB_ERR_INVALID_ARGUMENT, "linear_int8: types %d, %d, %d", p->x_dtype, p->out_dtype, p->bias_dtype);
  if (p->bias != nullptr && p->bias_dtype != FDB_FP32 && p->bias_dtype != p->out_dtype)
    return fail(FDB_ERR_INVALID_ARGUMENT, "linear_int8: the bias is of the output's type or fp32");
  if (p->rows < 0 || p->in_features <= 0 || p->out_features <= 0)
    return fail(FDB_ERR_INVALID_ARGUMENT, "linear_int8: %lld rows, %d -> %d features", (long long)p->rows, p->in_features, p->out_features);
  if (p->rows > (int64_t(1) << 31) - 512 || p->in_features > 131071 || p->out_features > (1 << 30))
    return fail(FDB_ERR_LIMIT, "linear_int8: %lld rows, %d -> %d features (an int32 sum holds 131071 products)", (long long)p->rows, p->in_features, p->out_features);
  return FDB_OK;
}

}  // namespace
}  // namespace fdb

using namespace fdb;

extern "C" FDB_API uint64_t fdb_linear_int8_workspace_bytes(const fdb_linear_int8_params* p) {
  clear_error();
  if (validate_int8(p) != FDB_OK || p->x_dtype == FDB_INT8 || p->rows == 0 || int8_is_small(*p)) return 0;
  return rows_bytes(*p) + uint64_t(p->rows) * sizeof(float);
}

extern "C" FDB_API int fdb_linear_int8(const fdb_linear_int8_params* p, void* stream) {
  clear_error();
  int rc = validate_int8(p);
  if (rc != FDB_OK) return rc;
  const bool given = p->x_dtype == FDB_INT8;
  if (p->x == nullptr || p->weight == nullptr || p->weight_scale == nullptr || p->out == nullptr || (given && p->x_scale == nullptr))
    return fail(FDB_ERR_INVALID_ARGUMENT, "linear_int8: x, weight, their scales and out must not be NULL");
  if (p->weight_pitch < p->in_features || (given && p->x_pitch < p->in_features))
    return fail(FDB_ERR_INVALID_ARGUMENT, "linear_int8: rows shorter than %d features", p->in_features);
  if (!aligned_to(16, p->weight) || p->weight_pitch % 16 != 0 || (given && (!aligned_to(16, p->x) || p->x_pitch % 16 != 0)))
    return fail(FDB_ERR_ALIGNMENT, "linear_int8: rows of integers must start on 16 bytes");
  if (!aligned_to(4, p->x_scale, p->weight_scale, p->status) || !aligned_to(type_bytes(p->out_dtype), p->out) ||
      (p->bias != nullptr && !aligned_to(type_bytes(p->bias_dtype), p->bias)) || (!given && !aligned_to(type_bytes(p->x_dtype), p->x)))
    return fail(FDB_ERR_ALIGNMENT, "linear_int8: tensors must be aligned to their elements");
  if (p->rows == 0) return FDB_OK;
  if (int8_is_small(*p)) return launch_linear_int8_small(*p, stream);
  const void* x = p->x;
  const float* x_scale = p->x_scale;
  int64_t pitch = p->x_pitch;
  if (!given) {
    const uint64_t need = rows_bytes(*p) + uint64_t(p->rows) * sizeof(float);
    if (p->workspace == nullptr || p->workspace_bytes < need || !aligned_to(256, p->workspace))
      return fail(FDB_ERR_WORKSPACE, "linear_int8: workspace of %llu bytes needed (256-byte aligned), %llu given", (unsigned long long)need,
                  (unsigned long long)p->workspace_bytes);
    float* scale = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + rows_bytes(*p));
    pitch = pitch_of(*p);
    if ((rc = launch_quantize_int8(p->x, p->x_dtype, p->rows, p->in_features, p->workspace, pitch, scale, stream)) != FDB_OK) return rc;
    x = p->workspace;
    x_scale = scale;
  }
  const int sms = sm_count();
  if (sms <= 0) return fail(FDB_ERR_CUDA, "linear_int8 set-up: no device");
  const Config* best = nullptr;
  int64_t best_cost = 0, best_tiles = 0;
  for (const Config& f : kConfigs) {
    const int64_t tiles = (p->rows + kBM * f.cg - 1) / (kBM * f.cg) * ((p->out_features + f.bn - 1) / f.bn);
    const int64_t units = sms / f.cg, waves = (tiles + units - 1) / units;
    const int64_t loop = (int64_t)((p->in_features + kBK - 1) / kBK) * f.clocks, epilogue = p->gelu != 0 ? f.epilogue * 9 / 5 : f.epilogue;
    const int64_t cost = waves * std::max(loop, epilogue) + std::min(loop, epilogue);
    if (best == nullptr || cost < best_cost) { best = &f; best_cost = cost; best_tiles = tiles; }
  }
  if (best_tiles * 2 > 2147483647LL) return fail(FDB_ERR_LIMIT, "linear_int8: %lld rows x %d features", (long long)p->rows, p->out_features);
  Int8Args a;
  rc = make_map_bytes(&a.tm_x, x, p->rows, p->in_features, pitch, kBM, "x");
  if (rc == FDB_OK) rc = make_map_bytes(&a.tm_w, p->weight, p->out_features, p->in_features, p->weight_pitch, best->bn / best->cg, "weight");
  if (rc != FDB_OK) return rc;
  a.x_scale = x_scale; a.w_scale = p->weight_scale; a.bias = p->bias; a.out = p->out; a.status = p->status;
  a.rows = p->rows; a.k = p->in_features; a.n = p->out_features;
  a.tiles_n = (p->out_features + best->bn - 1) / best->bn;
  a.bias_fp32 = p->bias_dtype == FDB_FP32;
  a.wide = p->out_features * (int64_t)type_bytes(p->out_dtype) % 16 == 0 && aligned_to(16, p->out, p->weight_scale, p->bias);
  if (a.wide) {
    const CUtensorMapDataType type = p->out_dtype == FDB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                              : (p->out_dtype == FDB_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32);
    rc = make_map_out(&a.tm_out, p->out, p->rows, p->out_features, type, (int)type_bytes(p->out_dtype), 32, "out");
    if (rc != FDB_OK) return rc;
  }
  const int units = sms / best->cg;
  const int grid = (int)(best_tiles < units ? best_tiles : units) * best->cg;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool gelu = p->gelu != 0, chained = !given;
#define FDB_INT8_TILE(CG, BN, COLS) launch_type<CG, BN, COLS>(a, grid, p->out_dtype, gelu, chained, s)
  if (best->bn == 256) return best->cols == 128 ? FDB_INT8_TILE(2, 256, 128) : FDB_INT8_TILE(2, 256, 64);
  if (best->cg == 2) return FDB_INT8_TILE(2, 128, 32);
  return best->bn == 128 ? FDB_INT8_TILE(1, 128, 32) : FDB_INT8_TILE(1, 64, 32);
#undef FDB_INT8_TILE
}
