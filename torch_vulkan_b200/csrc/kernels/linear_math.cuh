// Activations of the fused linear layer and their derivatives, in float32.
//   gelu       z Phi(z) = 0.5 z (1 + erf(z / sqrt 2))
//   gelu_tanh  0.5 z (1 + tanh u), u = sqrt(2 / pi) (z + 0.044715 z^3): the same as z / (1 + exp(-2 u)), which takes one
//              exponential and keeps its relative accuracy where 1 + tanh u would cancel
//   silu       z / (1 + exp(-z))
// Phi for 16-bit results: with t = 1 / (1 + 0.36 |z|), Phi(-|z|) = exp(-z^2 / 2) t P(t), P of degree 6, fitted by weighted least
// squares to erfcx for the least relative error (6.3e-7 for |z| <= 12). It takes about half of the instructions of 1 + erf, keeps
// its relative accuracy in the tail where that sum cancels, and the exponential is the one that the derivative needs as well.
// FAST (results that are rounded to 16 bits): the exponential and the division are the hardware's approximations, a few
// units of 2^-22 off, 2^-11 of the rounding of a float16 that follows. Float32 results take the library's functions.
#pragma once

#include <cuda_runtime.h>

#include "tvb200.h"

namespace tvb {

constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f, kSqrtHalf = 0.7071067811865476f, kInvSqrt2Pi = 0.3989422804014327f;

template <bool FAST>
__device__ __forceinline__ float sigmoid_f(float v) {
  if (FAST) return __fdividef(1.0f, 1.0f + __expf(-v));
  return 1.0f / (1.0f + expf(-v));
}

template <bool FAST>
__device__ __forceinline__ float gate_f(float z, float v) {  // z * sigmoid(v)
  if (FAST) return __fdividef(z, 1.0f + __expf(-v));
  return z / (1.0f + expf(-v));
}

// Phi(z); *density receives exp(-z^2 / 2).
__device__ __forceinline__ float phi_fast(float z, float* density) {
  const float a = fabsf(z), e = __expf(-0.5f * z * z), t = __fdividef(1.0f, fmaf(0.36f, a, 1.0f));
  float q = 0.0479438306f;
  q = fmaf(q, t, -0.182800836f);
  q = fmaf(q, t, 0.18508936f);
  q = fmaf(q, t, 0.0236945049f);
  q = fmaf(q, t, 0.140766829f);
  q = fmaf(q, t, 0.141579752f);
  q = fmaf(q, t, 0.143726872f);
  q *= t * e;
  *density = e;
  return z < 0.0f ? q : 1.0f - q;
}

template <bool FAST>
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case TVB_ACT_RELU: return z < 0.0f ? 0.0f : z;  // (a NaN stays one)
    case TVB_ACT_GELU: {
      float e;
      return FAST ? z * phi_fast(z, &e) : 0.5f * z * (1.0f + erff(z * kSqrtHalf));
    }
    case TVB_ACT_GELU_TANH: return gate_f<FAST>(z, 2.0f * kGeluC * (z + kGeluA * z * z * z));
    case TVB_ACT_SILU: return gate_f<FAST>(z, z);
    default: return z;
  }
}

template <bool FAST>
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case TVB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case TVB_ACT_GELU: {
      if (FAST) {
        float e;
        const float c = phi_fast(z, &e);
        return fmaf(z * kInvSqrt2Pi, e, c);
      }
      return 0.5f * (1.0f + erff(z * kSqrtHalf)) + z * expf(-0.5f * z * z) * kInvSqrt2Pi;
    }
    case TVB_ACT_GELU_TANH: {  // with s = sigmoid(2 u): s + z s (1 - s) 2 u'
      const float z2 = z * z;
      const float s = sigmoid_f<FAST>(2.0f * kGeluC * z * (1.0f + kGeluA * z2));
      return s + z * s * (1.0f - s) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * z2);
    }
    case TVB_ACT_SILU: {
      const float s = sigmoid_f<FAST>(z);
      return s + z * s * (1.0f - s);
    }
    default: return 1.0f;
  }
}

}  // namespace tvb
