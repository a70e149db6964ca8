// Activations of the linear products and their derivatives, in float32.
#pragma once

#include <cuda_runtime.h>

#include "../../include/kda_b200.h"

namespace kda {

// Phi(z), the standard normal distribution function, and e^{-z^2/2}.  With t = 1 / (1 + p |z| / sqrt 2)
// the lower tail is Phi(-|z|) = e^{-z^2/2} t (c0 + c1 t + .. + c5 t^5): a polynomial in t for
// erfcx(x) / 2 = e^{x^2} erfc(x) / 2 as in the classical rational approximations of erfc, with
// p = 0.45 and coefficients fitted here (least squares reweighted to the smallest largest
// relative error on x in [0, 9.5]): 9.0e-6 relative everywhere, the tail included, a fiftieth of half
// a step of the 16-bit results.  Two special-function operations (reciprocal, exponential).
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  const float t = __fdividef(1.f, fmaf(fabsf(z), 0.31819805153394637f, 1.f));
  e = exp2f(z * z * -0.72134752044448170f);
  float q = fmaf(t, -0.06728928729849852f, 0.14410881126505157f);
  q = fmaf(t, q, 0.0471456132106681f);
  q = fmaf(t, q, 0.122865324257533f);
  q = fmaf(t, q, 0.12621719678818977f);
  q = fmaf(t, q, 0.1269478731670778f);
  const float h = q * t * e;
  return z < 0.f ? h : 1.f - h;
}
__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

constexpr float kTanhA = 1.5957691216057308f;  // 2 sqrt(2 / pi): 1 + tanh(u) = 2 logistic(2 u)
constexpr float kTanhB = 0.044715f;

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case KDA_ACT_RELU: return z < 0.f ? 0.f : z;  // a NaN stays one
    case KDA_ACT_SILU: return z * logistic(z);
    case KDA_ACT_GELU: {
      float e;
      return z * normal_cdf(z, e);
    }
    case KDA_ACT_GELU_TANH: return z * logistic(kTanhA * z * fmaf(kTanhB, z * z, 1.f));
    default: return z;
  }
}
__device__ __forceinline__ float activate_grad(int act, float z) {
  switch (act) {
    case KDA_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case KDA_ACT_SILU: {
      const float s = logistic(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    case KDA_ACT_GELU: {
      float e;
      const float c = normal_cdf(z, e);
      return fmaf(z * 0.3989422804014327f, e, c);
    }
    case KDA_ACT_GELU_TANH: {
      const float s = logistic(kTanhA * z * fmaf(kTanhB, z * z, 1.f));
      return fmaf(z * s * (1.f - s), kTanhA * fmaf(3.f * kTanhB, z * z, 1.f), s);
    }
    default: return 1.f;
  }
}

}  // namespace kda
