// Activations of the expert products and their slopes, in fp32.
//   relu  z < 0 ? 0 : z                slope 1 where z > 0
//   gelu  z Phi(z)                     slope Phi(z) + z phi(z)
//   silu  z s(z), s(z) = 1 / (1 + exp(-z))      slope s(z) + z s(z) (1 - s(z))
// Phi(-|z|) = phi-shaped factor exp(-z^2 / 2) times the slowly varying erfcx(|z| / sqrt 2) / 2.  The second
// factor behaves like 1 / |z| far out, so with t = 1 / (1 + 0.26 |z|) it is t times a polynomial in t:
// degree 8, the coefficients a reweighted least-squares fit of the relative error over 0 <= |z| <= 14.5
// (at most 2.9e-8; beyond, exp(-z^2 / 2) is zero in fp32).  Evaluated in fp32 the absolute error of Phi is
// at most 2.4e-7 and its relative error 4e-6 out to z = -9, nearly all of that from the rounding of the exponent 0.72 z^2 (with an exact
// exponential it is 4.2e-7).  One reciprocal, one exponential and no branch: the
// library's erfcf made the activation, not the product, the longest part of a tile (452 us against
// 239 us for the product alone at 16 x 2,048 rows, K = N = 2,048).
// Far out, where the formulas would multiply an infinity with a zero, the limits are taken; NaN stays NaN.
#pragma once

#include "asp_internal.h"

namespace asp {

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.44269504f;

// Phi(z); *e receives exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float* e) {
  const float t = rcp_fast(fmaf(0.26f, fabsf(z), 1.f));
  float q = 0.0302303012f;
  q = fmaf(q, t, -0.151494438f);
  q = fmaf(q, t, 0.248733209f);
  q = fmaf(q, t, -0.147789338f);
  q = fmaf(q, t, 0.158758764f);
  q = fmaf(q, t, 0.0519648210f);
  q = fmaf(q, t, 0.102788682f);
  q = fmaf(q, t, 0.103050974f);
  q = fmaf(q, t, 0.103757022f);
  *e = exp2_fast((-0.5f * kLog2e) * (z * z));
  const float below = q * t * *e;
  return z < 0.f ? below : 1.f - below;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == ALPHASPARSE_ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == ALPHASPARSE_ACT_GELU) {
    float e;
    z = z < -20.f ? -20.f : z;
    return z * normal_cdf(z, &e);
  }
  if constexpr (ACT == ALPHASPARSE_ACT_SILU) {
    z = z < -120.f ? -120.f : z;
    return z * rcp_fast(1.f + exp2_fast(-kLog2e * z));
  }
  return z;
}

// Two values at once, for kernels whose arithmetic counts: packed pairs take one instruction for two multiply-adds, each with the
// rounding of the scalar form.  The two values share instructions, never operands: they are rows of different tokens (the second may
// be a row behind the last segment), and a row's bits may not depend on its neighbour's.  So each takes a reciprocal of its own.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }

template <int ACT>
__device__ __forceinline__ void activate2(float& z0, float& z1) {
  if constexpr (ACT == ALPHASPARSE_ACT_GELU) {
    const float a0 = fminf(fabsf(z0), 20.f), a1 = fminf(fabsf(z1), 20.f);
    const uint64_t az = pack2(a0, a1);
    float d0, d1;
    unpack2(fma2(az, both(0.26f), both(1.f)), d0, d1);
    const uint64_t t = pack2(rcp_fast(d0), rcp_fast(d1));
    uint64_t q = both(0.0302303012f);
    q = fma2(q, t, both(-0.151494438f));
    q = fma2(q, t, both(0.248733209f));
    q = fma2(q, t, both(-0.147789338f));
    q = fma2(q, t, both(0.158758764f));
    q = fma2(q, t, both(0.0519648210f));
    q = fma2(q, t, both(0.102788682f));
    q = fma2(q, t, both(0.103050974f));
    q = fma2(q, t, both(0.103757022f));
    float x0, x1, p0, p1;
    unpack2(mul2(mul2(az, az), both(-0.5f * kLog2e)), x0, x1);
    unpack2(mul2(mul2(q, t), pack2(exp2_fast(x0), exp2_fast(x1))), p0, p1);
    z0 = z0 < -20.f ? 0.f : z0 * (z0 < 0.f ? p0 : 1.f - p0);
    z1 = z1 < -20.f ? 0.f : z1 * (z1 < 0.f ? p1 : 1.f - p1);
  } else {
    z0 = activate<ACT>(z0);
    z1 = activate<ACT>(z1);
  }
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == ALPHASPARSE_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == ALPHASPARSE_ACT_GELU) {
    float e;
    z = z < -20.f ? -20.f : z > 20.f ? 20.f : z;
    const float p = normal_cdf(z, &e);
    return fmaf(z, 0.398942280f * e, p);
  }
  if constexpr (ACT == ALPHASPARSE_ACT_SILU) {
    z = z < -120.f ? -120.f : z > 120.f ? 120.f : z;
    // e = exp(-|z|) in (0, 1]: s(z) (1 - s(z)) = e / (1 + e)^2 is symmetric in z
    const float e = exp2_fast(-kLog2e * fabsf(z)), r = rcp_fast(1.f + e), er = e * r;
    return fmaf(z, er * r, z < 0.f ? er : r);
  }
  return 1.f;
}

}  // namespace asp
