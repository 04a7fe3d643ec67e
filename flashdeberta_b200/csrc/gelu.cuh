// GELU(v) = v * Phi(v) with Phi from the complementary error function in the rational form of Abramowitz & Stegun 7.1.26
// (absolute error 1.5e-7, far below half a bf16 ulp of the result): one reciprocal, one exponential and nine FMAs per
// element, about half of what erff costs — with erff the epilogue of the linear kernel would be longer than its main loop.
#pragma once

#include "sm100_ptx.cuh"

namespace fdb {

// v * Phi(v) with Phi(v) = 1/2 erfc(-v / sqrt 2):  v * Phi(v) = v / 2 + |v| * (1/2 - q),  q = 1/2 erfc(|v| / sqrt 2), for a pair.
// Two-wide forms where they exist: a third fewer instructions beside a main loop that is bound by power at large sizes
// (16384 x 768 -> 3072: 75.8 -> 74.7 us, against 63 us without the activation).
__device__ __forceinline__ uint64_t gelu_erf2(uint64_t v) {
  const uint64_t av = v & 0x7fffffff7fffffffull;
  const uint64_t z = ptx::mul_f32x2(av, ptx::pack_f32x2(0.70710678118654752f, 0.70710678118654752f));
  float d0, d1, e0, e1, t0, t1;
  ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(0.3275911f, 0.3275911f), z, ptx::pack_f32x2(1.f, 1.f)), d0, d1);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(d0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(d1));
  ptx::unpack_f32x2(ptx::mul_f32x2(ptx::mul_f32x2(z, z), ptx::pack_f32x2(-1.4426950408889634f, -1.4426950408889634f)), e0, e1);
  const uint64_t e = ptx::pack_f32x2(ptx::ex2(e0), ptx::ex2(e1)), t = ptx::pack_f32x2(t0, t1);
  auto both = [](float c) { return ptx::pack_f32x2(c, c); };
  uint64_t p = ptx::fma_f32x2(both(-0.5f * 1.061405429f), t, both(-0.5f * -1.453152027f));  // negated: h = 1/2 - p t e below
  p = ptx::fma_f32x2(p, t, both(-0.5f * 1.421413741f));
  p = ptx::fma_f32x2(p, t, both(-0.5f * -0.284496736f));
  p = ptx::fma_f32x2(p, t, both(-0.5f * 0.254829592f));
  const uint64_t h = ptx::fma_f32x2(ptx::mul_f32x2(p, t), e, both(0.5f));
  return ptx::fma_f32x2(av, h, ptx::mul_f32x2(v, both(0.5f)));
}

// The same for results in fp16 or bf16 whose values far below zero count: 1/2 erfc(z) = t P(t) e^(-z^2) with t = 1 / (1 + p z) and P, of
// degree 5, fitted here for the smallest relative error over 0 <= z <= 12 (8.9e-6), and v Phi(v) = max(v, 0) - |v| 1/2 erfc(|v| / sqrt 2),
// which loses nothing where Phi(v) is small.  With the exponential's argument rounded 1.8e-5 at v = -13, where the result leaves fp32's
// range: a twenty-seventh of fp16's half step, a two hundredth of bf16's.  +inf stays, -inf gives zero, NaN stays.
__device__ __forceinline__ uint64_t gelu_tail2(uint64_t v) {
  auto both = [](float c) { return ptx::pack_f32x2(c, c); };
  float v0, v1, d0, d1, e0, e1, t0, t1, r0, r1;
  ptx::unpack_f32x2(v, v0, v1);
  const uint64_t a = ptx::pack_f32x2(fminf(fabsf(v0), 1e4f), fminf(fabsf(v1), 1e4f));  // (an infinity times zero would be a NaN)
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r0) : "f"(v0));
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r1) : "f"(v1));
  ptx::unpack_f32x2(ptx::fma_f32x2(a, both(0.65f * 0.70710678118654752f), both(1.f)), d0, d1);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(d0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(d1));
  ptx::unpack_f32x2(ptx::mul_f32x2(ptx::mul_f32x2(a, both(-0.5f * 1.4426950408889634f)), a), e0, e1);
  const uint64_t e = ptx::pack_f32x2(ptx::ex2(e0), ptx::ex2(e1)), t = ptx::pack_f32x2(t0, t1);
  uint64_t p = ptx::fma_f32x2(both(-0.0718298222776901f), t, both(0.23586562590151855f));  // -P: what is taken off
  p = ptx::fma_f32x2(p, t, both(-0.17785580337148693f));
  p = ptx::fma_f32x2(p, t, both(-0.1160826767118539f));
  p = ptx::fma_f32x2(p, t, both(-0.18690448711125093f));
  p = ptx::fma_f32x2(p, t, both(-0.1831955746192981f));
  return ptx::fma_f32x2(ptx::mul_f32x2(a, e), ptx::mul_f32x2(p, t), ptx::pack_f32x2(r0, r1));
}

// And for results in fp32, where every one of these roundings would show: P of degree 9 (fitted over 0 <= z <= 9.4, 0.11 * 2^-24), and the
// exponential's argument in two parts, what |v|^2 and its product with log2(e) / 2 lose by their rounding put back behind it.  With a
// correct reciprocal and exponential every step in fp32 leaves 5.8 * 2^-24 of |v| 1/2 erfc(|v| / sqrt 2); the approximate ones may add
// 2 and 4.  Below v = -13.2 the exponential is out of its range: zero, where the result would be below 2^-126.  (CUDA's erfcf in its
// place: 16384 x 1024 -> 4096 155 us, the largest relative error in v > -4 3.0e-7; these steps 92 us and 4.0e-7; gelu_tail2's
// with degree 6 83 us and 1.4e-6; 0.5 v erfcf(-v / sqrt 2) of a rounded argument 1.1e-6.)
__device__ __forceinline__ uint64_t gelu_fine2(uint64_t v) {
  auto both = [](float c) { return ptx::pack_f32x2(c, c); };
  constexpr uint64_t kSigns = 0x8000000080000000ull;
  float v0, v1, d0, d1, e0, e1, t0, t1, r0, r1;
  ptx::unpack_f32x2(v, v0, v1);
  const uint64_t a = ptx::pack_f32x2(fminf(fabsf(v0), 1e4f), fminf(fabsf(v1), 1e4f));  // (an infinity times zero would be a NaN)
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r0) : "f"(v0));
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r1) : "f"(v1));
  ptx::unpack_f32x2(ptx::fma_f32x2(a, both(0.55f * 0.70710678118654752f), both(1.f)), d0, d1);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(d0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(d1));
  const uint64_t square = ptx::mul_f32x2(a, a), square_low = ptx::fma_f32x2(a, a, square ^ kSigns);
  constexpr float kHalfLog2e = 0.72134752044448170f, kHalfLog2eLow = 0.72134752044448170 - (double)kHalfLog2e;
  const uint64_t high = ptx::mul_f32x2(square, both(-kHalfLog2e));
  uint64_t low = ptx::fma_f32x2(square, both(-kHalfLog2e), high ^ kSigns);
  low = ptx::fma_f32x2(square, both(-kHalfLog2eLow), low);
  low = ptx::fma_f32x2(square_low, both(-kHalfLog2e), low);
  ptx::unpack_f32x2(high, e0, e1);
  uint64_t e = ptx::pack_f32x2(ptx::ex2(e0), ptx::ex2(e1));
  e = ptx::fma_f32x2(e, ptx::mul_f32x2(low, both(0.69314718055994531f)), e);
  const uint64_t t = ptx::pack_f32x2(t0, t1);
  uint64_t p = ptx::fma_f32x2(both(-0.02902292087674141f), t, both(0.16832473874092102f));  // -P: what is taken off
  p = ptx::fma_f32x2(p, t, both(-0.39061447978019714f));
  p = ptx::fma_f32x2(p, t, both(0.42670324444770813f));
  p = ptx::fma_f32x2(p, t, both(-0.18197107315063477f));
  p = ptx::fma_f32x2(p, t, both(0.04749220609664917f));
  p = ptx::fma_f32x2(p, t, both(-0.10102356225252151f));
  p = ptx::fma_f32x2(p, t, both(-0.12941037118434906f));
  p = ptx::fma_f32x2(p, t, both(-0.15533173084259033f));
  p = ptx::fma_f32x2(p, t, both(-0.1551460474729538f));
  return ptx::fma_f32x2(ptx::mul_f32x2(a, e), ptx::mul_f32x2(p, t), ptx::pack_f32x2(r0, r1));
}

}  // namespace fdb
