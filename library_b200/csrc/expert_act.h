// Activations of the expert products and their slopes, in fp32.
//   relu  z > 0 ? z : 0                slope 1 where z > 0
//   gelu  z Phi(z) = z erfc(-z / sqrt 2) / 2    slope Phi(z) + z phi(z)
//   silu  z s(z), s(z) = 1 / (1 + exp(-z))      slope s(z) + z s(z) (1 - s(z))
// erfc keeps the relative accuracy of Phi(z) for negative z, where 1 + erf would cancel.  Far out,
// where the formulas would multiply an infinity with a zero, the limits are taken.
#pragma once

#include "asp_internal.h"

namespace asp {

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == ALPHASPARSE_ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == ALPHASPARSE_ACT_GELU) return z < -20.f ? 0.f : 0.5f * z * erfcf(-0.70710678f * z);
  if constexpr (ACT == ALPHASPARSE_ACT_SILU) return z < -110.f ? 0.f : __fdividef(z, 1.f + expf(-z));
  return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == ALPHASPARSE_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == ALPHASPARSE_ACT_GELU) {
    if (fabsf(z) > 20.f) return z > 0.f ? 1.f : 0.f;
    return 0.5f * erfcf(-0.70710678f * z) + z * (0.39894228f * expf(-0.5f * z * z));
  }
  if constexpr (ACT == ALPHASPARSE_ACT_SILU) {
    if (fabsf(z) > 110.f) return z > 0.f ? 1.f : 0.f;
    // e = exp(-|z|) in (0, 1]: s(z) (1 - s(z)) = e / (1 + e)^2 is symmetric in z
    const float e = expf(-fabsf(z)), r = __fdividef(1.f, 1.f + e);
    return (z >= 0.f ? r : e * r) + z * (e * r * r);
  }
  return 1.f;
}

}  // namespace asp
