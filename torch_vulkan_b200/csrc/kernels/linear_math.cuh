// Activations of the fused linear layer and their derivatives, in float32.
//   gelu       z Phi(z) = 0.5 z (1 + erf(z / sqrt 2))
//   gelu_tanh  0.5 z (1 + tanh u), u = sqrt(2 / pi) (z + 0.044715 z^3): the same as z / (1 + exp(-2 u)), which takes one
//              exponential and keeps its relative accuracy where 1 + tanh u would cancel
//   silu       z / (1 + exp(-z))
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

template <bool FAST>
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case TVB_ACT_RELU: return z < 0.0f ? 0.0f : z;  // (a NaN stays one)
    case TVB_ACT_GELU: return 0.5f * z * (1.0f + erff(z * kSqrtHalf));
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
      const float e = FAST ? __expf(-0.5f * z * z) : expf(-0.5f * z * z);
      return 0.5f * (1.0f + erff(z * kSqrtHalf)) + z * e * kInvSqrt2Pi;
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
