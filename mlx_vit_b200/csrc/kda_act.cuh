// Activations of the linear products and their derivatives, in float32.
#pragma once

#include <cuda_runtime.h>

#include "../../include/kda_b200.h"

namespace kda {

// Two float32 operations in one instruction (sm_100's packed forms).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.ftz.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.ftz.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.ftz.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// The standard normal's lower tail h = Phi(-|z|) and e = e^{-z^2/2}: h = e q(|z|) with
// q(x) = e^{x^2/2} Phi(-x), which falls smoothly from 1/2 to 0.08 on [0, 4.95] and is a polynomial of
// degree 9 in x - 2.475 there, fitted here to the smallest largest relative error (least squares
// reweighted): 3.0e-5, evaluation included, a sixteenth of half a step of fp16.  Beyond 4.95
// (x is cut there) h is below 4e-7 and z h off by 2e-9 at most.  One special-function operation an
// element and packed products: a form with a reciprocal and six products instead took twice the
// issue slots and made the epilogue, not the tensor cores, the bound of short sums.
__device__ __forceinline__ float2 normal_tail(float2 z, float2 &x, float2 &e) {
  x = make_float2(fminf(fabsf(z.x), 4.95f), fminf(fabsf(z.y), 4.95f));
  const float2 w = mul2(mul2(z, z), both(-0.72134752044448170f));
  e = make_float2(exp2f(w.x), exp2f(w.y));
  const float2 u = add2(x, both(-2.475f));
  float2 q = fma2(both(-1.3505667766366969e-06f), u, both(7.080250270519173e-06f));
  q = fma2(q, u, both(-1.2636107385333162e-05f));
  q = fma2(q, u, both(4.3477630242705345e-05f));
  q = fma2(q, u, both(-0.00026864901883527637f));
  q = fma2(q, u, both(0.0010978090576827526f));
  q = fma2(q, u, both(-0.003940265160053968f));
  q = fma2(q, u, both(0.013904363848268986f));
  q = fma2(q, u, both(-0.046298861503601074f));
  q = fma2(q, u, both(0.14248423278331757f));
  return mul2(q, e);
}
__device__ __forceinline__ float2 gelu2(float2 z) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
  float2 x, e;
  const float2 h = normal_tail(z, x, e);
  return fma2(make_float2(-x.x, -x.y), h, make_float2(fmaxf(z.x, 0.f), fmaxf(z.y, 0.f)));
}
__device__ __forceinline__ float2 gelu_grad2(float2 z) {  // Phi(z) + z phi(z)
  float2 x, e;
  const float2 h = normal_tail(z, x, e);
  const float2 c = make_float2(z.x < 0.f ? h.x : 1.f - h.x, z.y < 0.f ? h.y : 1.f - h.y);
  return fma2(mul2(z, both(0.3989422804014327f)), e, c);
}
__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

constexpr float kTanhA = 1.5957691216057308f;  // 2 sqrt(2 / pi): 1 + tanh(u) = 2 logistic(2 u)
constexpr float kTanhB = 0.044715f;

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case KDA_ACT_RELU: return z < 0.f ? 0.f : z;  // a NaN stays one
    case KDA_ACT_SILU: return z * logistic(z);
    case KDA_ACT_GELU: return gelu2(both(z)).x;
    case KDA_ACT_GELU_TANH: return z * logistic(kTanhA * z * fmaf(kTanhB, z * z, 1.f));
    default: return z;
  }
}
__device__ __forceinline__ float activate_grad(int act, float z) {  // not ReLU's: grad_through
  switch (act) {
    case KDA_ACT_SILU: {
      const float s = logistic(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    case KDA_ACT_GELU: return gelu_grad2(both(z)).x;
    case KDA_ACT_GELU_TANH: {
      const float s = logistic(kTanhA * z * fmaf(kTanhB, z * z, 1.f));
      // s (1 - s) is zero from |z| = 11 on, where z^2 may be infinite: cut far behind that
      return fmaf(z * s * (1.f - s), kTanhA * fmaf(3.f * kTanhB, fminf(z * z, 1e6f), 1.f), s);
    }
    default: return 1.f;
  }
}

// two at once
__device__ __forceinline__ float2 activate2(int act, float2 z) {
  if (act == KDA_ACT_GELU) return gelu2(z);
  return make_float2(activate(act, z.x), activate(act, z.y));
}
// A gradient g at an activation's result to the one at its input z: g act'(z).  ReLU's selects, as torch's:
// behind a dead unit an infinite or NaN g is dropped, and where z is NaN it passes.
__device__ __forceinline__ float grad_through(int act, float g, float z) {
  if (act == KDA_ACT_RELU) return z <= 0.f ? 0.f : g;
  return g * activate_grad(act, z);
}
__device__ __forceinline__ float2 grad_through2(int act, float2 g, float2 z) {
  if (act == KDA_ACT_RELU) return make_float2(grad_through(act, g.x, z.x), grad_through(act, g.y, z.y));
  return mul2(g, act == KDA_ACT_GELU ? gelu_grad2(z) : make_float2(activate_grad(act, z.x), activate_grad(act, z.y)));
}

}  // namespace kda
