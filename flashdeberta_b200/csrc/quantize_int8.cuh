// The rounding of a row to 8-bit integers, as fdb_quantize_int8 defines it, for the kernels that do it: the largest magnitude of a row
// (compared as the bits of absolute values: a NaN is larger than everything there, so it reaches the scale), the scale, the integers.
#pragma once

#include "row_team.cuh"

namespace fdb {

// Largest magnitude of a thread's elements, as bits of T's absolute values; and such bits as fp32.
template <int V> __device__ __forceinline__ uint32_t top_of(const RowWords<float, V>& r) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < V * kRowElems; ++j) top = max(top, r.w[j] & 0x7fffffffu);
  return top;
}
template <typename T, int V> __device__ __forceinline__ uint32_t top_of(const RowWords<T, V>& r) {  // two at a time
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < V * kRowElems / 2; ++j) top = __vmaxu2(top, r.w[j] & 0x7fff7fffu);
  return max(top & 0xffffu, top >> 16);
}
template <typename T> __device__ __forceinline__ float bits_to_float(uint32_t b) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(b);
  const unsigned short h = (unsigned short)b;
  return to_float<T>(*reinterpret_cast<const T*>(&h));
}

// Four products with the reciprocal scale, each rounded to fp32 and then to a whole number, as bytes: 1.5 * 2^23 added, the number is in
// the lowest bits.  (float-to-int conversions run at a quarter of the rate.)
__device__ __forceinline__ uint32_t four_bytes(const float* v, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], inv), 12582912.f));  // (as one FMA the product would not be rounded)
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// What a row is scaled by.
struct Int8Scale { float scale, inv; bool finite; };
template <typename T> __device__ __forceinline__ Int8Scale int8_scale(uint32_t top_bits) {
  const float amax = bits_to_float<T>(top_bits);
  const bool zero = amax < 7.888609052e-31f, finite = amax <= 3.402823466e+38f;  // 2^-100: the reciprocal would leave fp32's range
  return {zero ? 0.f : amax / 127.f, zero || !finite ? 0.f : 127.f / amax, finite};
}

}  // namespace fdb
