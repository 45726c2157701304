// What a product's result goes through, and its derivative.  FAST, for results in bf16, whose own rounding is 2^-8 of the value: errors of 2^-19 of the value (of a slope
// near its zero: of 1) where |z| is up to 4, and beyond that those of e^x, whose argument is rounded to 2^-24 |x|: sigmoid, silu and their slopes 2^-20 at 12, 2^-18 at 87,
// tanh's slope twice that; gelu and its slope, of e^(-z^2 / 2), 2^-17 at -8, 2^-15 at -13.  Otherwise the library's functions and divisions.  A tile's epilogue has 128
// values a lane and nothing to hide their arithmetic behind: of the gradient through gelu (bf16 4096 x 8192, with dropout) a launch takes 80 us with the library's functions, 50 with these.
#pragma once
#include "common.h"

namespace cavs {

// e^x, 0 below 2^-126: the instruction of x log2 e, whose rounding is 2^-24 |x| of the result
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
// 1 / (1 + e^-z)
template <bool FAST>
__device__ __forceinline__ float logistic(float z) {
  if constexpr (!FAST) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + exp_fast(-z));
}
// e^-(z^2 / 2) and Phi(-|z|), the normal distribution: e^-(a^2) q(a) / 2, a = |z| / sqrt 2, q(a) = erfc(a) e^(a^2) as a polynomial of 1 / (1 + 0.6 a), fitted to
// 2e-8 of the value over 0 <= a <= 10.3 by weighted least squares at Chebyshev's points.  (Beyond a float holds nothing of it.)
__device__ __forceinline__ float normal_tail(float z, float *density) {
  const float a = fminf(fabsf(z), 14.5f) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(a, 0.6f, 1.f)), e = exp_fast(-a * a);
  float q = 0.045341771f;
  q = fmaf(q, t, -0.205804408f);
  q = fmaf(q, t, 0.29379943f);
  q = fmaf(q, t, 0.0312145744f);
  q = fmaf(q, t, -0.441048026f);
  q = fmaf(q, t, 0.236344293f);
  q = fmaf(q, t, 0.0677702501f);
  q = fmaf(q, t, 0.2980042696f);
  q = fmaf(q, t, 0.3356487155f);
  q = fmaf(q, t, 0.3387365341f);
  q = fmaf(q, t, -7.35271033e-6f);
  *density = e;
  return 0.5f * e * q;
}

template <bool FAST>
__device__ __forceinline__ float act_of(int act, float z) {
  switch (act) {
    case CAVS_ACT_RELU: return z < 0.f ? 0.f : z;
    case CAVS_ACT_TANH: {
      if constexpr (!FAST) return tanhf(z);
      const float e = exp_fast(-2.f * fabsf(z)), h = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e), u = z * z;
      const float near = z * fmaf(u, fmaf(u, fmaf(u, -0.0539682540f, 0.133333333f), -0.333333333f), 1.f);  // (the series: 4e-7 of the value at 1/4)
      return u < 0.0625f ? near : z == z ? copysignf(h, z) : z;
    }
    case CAVS_ACT_SIGMOID: return logistic<FAST>(z);
    case CAVS_ACT_SILU: return z * logistic<FAST>(z);
    case CAVS_ACT_GELU: {
      if constexpr (!FAST) return 0.5f * z * erfcf(-0.70710678f * z);
      float density;
      const float p = normal_tail(z, &density);
      return z * (z > 0.f ? 1.f - p : p);
    }
    default: return z;
  }
}
template <bool FAST>
__device__ __forceinline__ float slope_of(int act, float z) {
  switch (act) {
    case CAVS_ACT_RELU: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    case CAVS_ACT_TANH: {
      // (1 - tanh^2 = 4 e / (1 + e)^2, e = e^-2|z|: 1 - h of a tanh near 1 has lost what it is made of)
      const float e = FAST ? exp_fast(-2.f * fabsf(z)) : expf(-2.f * fabsf(z)), r = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
      return z == z ? 4.f * e * r * r : z;
    }
    case CAVS_ACT_SIGMOID: {
      const float g = logistic<FAST>(-fabsf(z));  // (even in z, and on this side 1 - g loses nothing)
      return g * (1.f - g);
    }
    case CAVS_ACT_SILU: {
      const float g = logistic<FAST>(z);
      return g * (1.f + z * (1.f - g));
    }
    case CAVS_ACT_GELU: {
      if constexpr (!FAST) return 0.5f * erfcf(-0.70710678f * z) + z * (0.39894228f * expf(-0.5f * z * z));
      float density;
      const float p = normal_tail(z, &density);
      return fmaf(z, 0.39894228f * density, z > 0.f ? 1.f - p : p);
    }
    default: return 1.f;
  }
}

}  // namespace cavs
