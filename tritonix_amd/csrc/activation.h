// Activations of a linear layer and their derivatives, in 32 bits.
#pragma once
#include "gemm_tile.h"

namespace tnx {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4 };

constexpr float GELU_C = 0.7978845608028654f;            // sqrt(2 / pi)
constexpr float GELU_A = 0.044715f;

// 1 / (1 + e^-z), from the reciprocal instruction: half its last bit off where the division would be exact, in 32 bits, at an eighth of the
// instructions
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// erfc(|z| / sqrt 2), and e = exp(-z^2 / 2) on the way: t P(t) e with t = 1 / (1 + p |z| / sqrt 2), as Hastings' rational approximations are formed.  P is of degree 7 and p 0.44, fitted
// here to the smallest largest error relative to the result, from 0 to |z| = 18 (weighted least squares, the weights raised where the error is largest, on 1200 Chebyshev points): 1.9e-7.
// In 32 bits (14 + 0.6 z^2) 2^-23 of the result, the exponential's argument being rounded.  A fit of five terms to the error itself, 1.5e-7 of it, is 2e-2 off relative to the
// result at |z| = 10, which gelu(-10) then is (4096 x 30000 x 768 bf16 with gelu: 281 us, with this 290; 8192 x 4096 x 4096 216 to 218 and 220).  A call of erff, with its branches,
// took 4096 x 14336 x 4096 with gelu 1.19 times the plain product's time, this 1.13.
__device__ __forceinline__ float erfc_abs(float z, float* e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.311126984f, __builtin_fabsf(z), 1.0f));      // p / sqrt 2
  float p = __builtin_fmaf(0.0715003982f, t, -0.279155076f);
  p = __builtin_fmaf(p, t, 0.298870951f);
  p = __builtin_fmaf(p, t, -0.0222975835f);
  p = __builtin_fmaf(p, t, 0.216995254f);
  p = __builtin_fmaf(p, t, 0.216934204f);
  p = __builtin_fmaf(p, t, 0.248935491f);
  p = __builtin_fmaf(p, t, 0.248216525f);
  *e = __builtin_amdgcn_exp2f(z * z * -0.721347520f);                                                 // log2(e) / 2
  return p * t * *e;
}

// gelu: z (1 + erf(z / sqrt 2)) / 2 is z q / 2 below zero and z - z q / 2 above, with q = erfc(|z| / sqrt 2): no cancellation next to -1.
// gelu_tanh: z (1 + tanh u) / 2 = z / (1 + e^-2u), which keeps its relative precision where tanh is next to -1
// The factor beside one that is zero in 32 bits past -128 (gelu's tail: past +-128) is held there, for the product of an infinity and a zero is no number: -inf gives zero and
// +inf itself.  (fmaxf and fminf take a NaN for the bound: the other factor is NaN then.)
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case ACT_RELU: return z <= 0.0f ? 0.0f : z;          // (a NaN stays one)
    case ACT_SILU: return fmaxf(z, -128.0f) * logistic(z);
    case ACT_GELU: {
      float e;
      const float half = 0.5f * fminf(fmaxf(z, -128.0f), 128.0f) * erfc_abs(z, &e);
      return z > 0.0f ? z - half : half;
    }
    case ACT_GELU_TANH: return fmaxf(z, -128.0f) * logistic(2.0f * GELU_C * (z + GELU_A * z * z * z));
    default: return z;
  }
}

// The derivative.  Past +-128 each is 0 or 1 in 32 bits, and held there: products of an infinity and a zero are no number.
__device__ __forceinline__ float activation_slope(float z, int act) {
  if (act == ACT_RELU) return z <= 0.0f ? 0.0f : z > 0.0f ? 1.0f : z;
  z = z > 128.0f ? 128.0f : z < -128.0f ? -128.0f : z;
  switch (act) {
    case ACT_SILU: {
      const float s = logistic(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case ACT_GELU: {
      float e;
      const float half = 0.5f * erfc_abs(z, &e);
      return (z > 0.0f ? 1.0f - half : half) + 0.3989422804014327f * z * e;
    }
    case ACT_GELU_TANH: {
      const float z2 = z * z, s = logistic(2.0f * GELU_C * z * (1.0f + GELU_A * z2));
      return s + 2.0f * z * s * (1.0f - s) * GELU_C * (1.0f + 3.0f * GELU_A * z2);
    }
    default: return 1.0f;
  }
}

}  // namespace tnx
