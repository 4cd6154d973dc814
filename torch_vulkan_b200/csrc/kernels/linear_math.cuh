// Activations of the fused linear layer and their derivatives, in float32.
//   gelu       z Phi(z) = 0.5 z (1 + erf(z / sqrt 2))
//   gelu_tanh  0.5 z (1 + tanh u), u = sqrt(2 / pi) (z + 0.044715 z^3): the same as z / (1 + exp(-2 u)), which takes one
//              exponential and keeps its relative accuracy where 1 + tanh u would cancel
//   silu       z / (1 + exp(-z))
// Float32 results take the library's functions, one value at a time. Results that are rounded to 16 bits take the forms on pairs
// below: the epilogue of a product has 64 clocks per output of a tile with 1024 values of r, and what it costs is instructions, so
// they work on two values at once wherever the hardware can, and take the exponential and the reciprocal from its
// approximations. Those are a few units of 2^-22 off, relative, and the exponent that goes in is itself rounded, which adds its size
// times 2^-24: 2^-18 for silu(-40), near 2^-17 at the far end of the tails. Half a step of the float16 that follows is 2^-11.
#pragma once

#include <cuda_runtime.h>

#include "ptx.cuh"
#include "tvb200.h"

namespace tvb {

constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f, kSqrtHalf = 0.7071067811865476f, kInvSqrt2Pi = 0.3989422804014327f;
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- float32 results

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case TVB_ACT_RELU: return z < 0.0f ? 0.0f : z;  // (a NaN stays one)
    case TVB_ACT_GELU: return 0.5f * z * (1.0f + erff(z * kSqrtHalf));
    case TVB_ACT_GELU_TANH: return z / (1.0f + expf(-2.0f * kGeluC * (z + kGeluA * z * z * z)));
    case TVB_ACT_SILU: return z / (1.0f + expf(-z));
    default: return z;
  }
}

// max(-most, min(z, most)), a NaN staying one. The derivatives take z so: from `most` on they are at their limits (0 or 1) in float32,
// and a z far beyond it, or an infinite one, would make them 0 times infinity.
__device__ __forceinline__ float within(float z, float most) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(most));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(-most));
  return z;
}
constexpr float kGeluMost = 30.0f, kSiluMost = 128.0f;

__device__ __forceinline__ float act_slope(float z, int act) {
  z = within(z, act == TVB_ACT_SILU ? kSiluMost : kGeluMost);
  switch (act) {
    case TVB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case TVB_ACT_GELU: return 0.5f * (1.0f + erff(z * kSqrtHalf)) + z * expf(-0.5f * z * z) * kInvSqrt2Pi;
    case TVB_ACT_GELU_TANH: {  // with s = sigmoid(2 u): s + z s (1 - s) 2 u'
      const float z2 = z * z;
      const float s = 1.0f / (1.0f + expf(-2.0f * kGeluC * z * (1.0f + kGeluA * z2)));
      return s + z * s * (1.0f - s) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * z2);
    }
    case TVB_ACT_SILU: {
      const float s = 1.0f / (1.0f + expf(-z));
      return s + z * s * (1.0f - s);
    }
    default: return 1.0f;
  }
}

// ---------------------------------------------------------------- 16-bit results, two values at a time

__device__ __forceinline__ uint64_t two(float v) { return ptx::both_f32x2(v); }

__device__ __forceinline__ uint64_t exp2_pair(uint64_t v) {
  float a, b;
  ptx::unpack_f32x2(v, a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  return ptx::pack_f32x2(__float_as_uint(a), __float_as_uint(b));
}

__device__ __forceinline__ uint64_t rcp_pair(uint64_t v) {
  float a, b;
  ptx::unpack_f32x2(v, a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return ptx::pack_f32x2(__float_as_uint(a), __float_as_uint(b));
}

// 1 / (1 + 2^v)
__device__ __forceinline__ uint64_t sigmoid2_pair(uint64_t v) { return rcp_pair(ptx::add_f32x2(exp2_pair(v), two(1.0f))); }

// max(z, 0), a NaN staying one
__device__ __forceinline__ uint64_t relu_pair(uint64_t z) {
  float a, b;
  ptx::unpack_f32x2(z, a, b);
  asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(a));
  asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(b));
  return ptx::pack_f32x2(__float_as_uint(a), __float_as_uint(b));
}

// min(|z|, 30): beyond it nothing below is distinguishable from its limit, and products with it stay finite
__device__ __forceinline__ uint64_t size_pair(uint64_t z) {
  float a, b;
  ptx::unpack_f32x2(z, a, b);
  a = fminf(fabsf(a), kGeluMost);
  b = fminf(fabsf(b), kGeluMost);
  return ptx::pack_f32x2(__float_as_uint(a), __float_as_uint(b));
}

__device__ __forceinline__ uint64_t within_pair(uint64_t z, float most) {
  float a, b;
  ptx::unpack_f32x2(z, a, b);
  return ptx::pack_f32x2(__float_as_uint(within(a, most)), __float_as_uint(within(b, most)));
}

// Phi(-a) for a >= 0; *density receives exp(-a^2 / 2). With t = 1 / (1 + 0.36 a), Phi(-a) = exp(-a^2 / 2) t P(t), P of degree 6,
// fitted by weighted least squares to erfcx for the least relative error (6.3e-7 for a <= 12 in exact arithmetic, 9.2e-7 with
// float32's roundings, to which the exponential adds its own): about half of the instructions of 1 + erf, accurate in the tail where that sum cancels, and the exponential is the one that the derivative needs as well.
__device__ __forceinline__ uint64_t tail_pair(uint64_t a, uint64_t* density) {
  const uint64_t e = exp2_pair(ptx::mul_f32x2(ptx::mul_f32x2(a, a), two(-0.5f * kLog2e)));
  const uint64_t t = rcp_pair(ptx::fma_f32x2(a, two(0.36f), two(1.0f)));
  uint64_t q = ptx::fma_f32x2(two(0.0479438306f), t, two(-0.182800836f));
  q = ptx::fma_f32x2(q, t, two(0.18508936f));
  q = ptx::fma_f32x2(q, t, two(0.0236945049f));
  q = ptx::fma_f32x2(q, t, two(0.140766829f));
  q = ptx::fma_f32x2(q, t, two(0.141579752f));
  q = ptx::fma_f32x2(q, t, two(0.143726872f));
  *density = e;
  return ptx::mul_f32x2(q, ptx::mul_f32x2(t, e));
}

template <int ACT>
__device__ __forceinline__ uint64_t act_pair(uint64_t z) {
  if constexpr (ACT == TVB_ACT_RELU) return relu_pair(z);
  if constexpr (ACT == TVB_ACT_GELU) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const uint64_t a = size_pair(z);
    uint64_t e;
    const uint64_t q = tail_pair(a, &e);
    return ptx::fma_f32x2(ptx::mul_f32x2(a, two(-1.0f)), q, relu_pair(z));
  }
  if constexpr (ACT == TVB_ACT_GELU_TANH) {
    const uint64_t u = ptx::fma_f32x2(ptx::mul_f32x2(z, z), two(-2.0f * kGeluC * kGeluA * kLog2e), two(-2.0f * kGeluC * kLog2e));
    return ptx::mul_f32x2(z, sigmoid2_pair(ptx::mul_f32x2(z, u)));
  }
  if constexpr (ACT == TVB_ACT_SILU) return ptx::mul_f32x2(z, sigmoid2_pair(ptx::mul_f32x2(z, two(-kLog2e))));
  return z;
}

template <int ACT>
__device__ __forceinline__ uint64_t slope_pair(uint64_t z) {
  if constexpr (ACT == TVB_ACT_RELU) {
    float a, b;
    ptx::unpack_f32x2(z, a, b);
    return ptx::pack_f32x2(a > 0.0f ? 0x3f800000u : 0u, b > 0.0f ? 0x3f800000u : 0u);
  }
  if constexpr (ACT == TVB_ACT_GELU) {  // Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi), Phi(z) = 0.5 + sign(z) (0.5 - Phi(-|z|))
    uint64_t e;
    z = within_pair(z, kGeluMost);
    const uint64_t q = tail_pair(size_pair(z), &e);
    float s0, s1, z0, z1;
    ptx::unpack_f32x2(ptx::fma_f32x2(q, two(-1.0f), two(0.5f)), s0, s1);
    ptx::unpack_f32x2(z, z0, z1);
    const uint64_t s = ptx::pack_f32x2(__float_as_uint(copysignf(s0, z0)), __float_as_uint(copysignf(s1, z1)));
    return ptx::fma_f32x2(ptx::mul_f32x2(z, two(kInvSqrt2Pi)), e, ptx::add_f32x2(s, two(0.5f)));
  }
  if constexpr (ACT == TVB_ACT_GELU_TANH) {  // with s = sigmoid(2 u): s + z s (1 - s) 2 u'
    z = within_pair(z, kGeluMost);
    const uint64_t z2 = ptx::mul_f32x2(z, z);
    const uint64_t u = ptx::fma_f32x2(z2, two(-2.0f * kGeluC * kGeluA * kLog2e), two(-2.0f * kGeluC * kLog2e));
    const uint64_t s = sigmoid2_pair(ptx::mul_f32x2(z, u));
    const uint64_t du = ptx::fma_f32x2(z2, two(6.0f * kGeluC * kGeluA), two(2.0f * kGeluC));
    const uint64_t rest = ptx::fma_f32x2(s, two(-1.0f), two(1.0f));
    return ptx::fma_f32x2(ptx::mul_f32x2(s, rest), ptx::mul_f32x2(z, du), s);
  }
  if constexpr (ACT == TVB_ACT_SILU) {
    z = within_pair(z, kSiluMost);
    const uint64_t s = sigmoid2_pair(ptx::mul_f32x2(z, two(-kLog2e)));
    const uint64_t rest = ptx::fma_f32x2(s, two(-1.0f), two(1.0f));
    return ptx::fma_f32x2(ptx::mul_f32x2(s, rest), z, s);
  }
  return two(1.0f);
}

// N pairs at once, the choice of activation made once for all of them.
template <int N>
__device__ __forceinline__ void activate_pairs(uint64_t (&v)[N], int act) {
  switch (act) {
    case TVB_ACT_RELU:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = act_pair<TVB_ACT_RELU>(v[e]);
      break;
    case TVB_ACT_GELU:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = act_pair<TVB_ACT_GELU>(v[e]);
      break;
    case TVB_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = act_pair<TVB_ACT_GELU_TANH>(v[e]);
      break;
    case TVB_ACT_SILU:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = act_pair<TVB_ACT_SILU>(v[e]);
      break;
    default: break;
  }
}

// v *= act'(z)
template <int N>
__device__ __forceinline__ void times_slope_pairs(uint64_t (&v)[N], const uint64_t (&z)[N], int act) {
  switch (act) {
    case TVB_ACT_RELU:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = ptx::mul_f32x2(v[e], slope_pair<TVB_ACT_RELU>(z[e]));
      break;
    case TVB_ACT_GELU:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = ptx::mul_f32x2(v[e], slope_pair<TVB_ACT_GELU>(z[e]));
      break;
    case TVB_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = ptx::mul_f32x2(v[e], slope_pair<TVB_ACT_GELU_TANH>(z[e]));
      break;
    case TVB_ACT_SILU:
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = ptx::mul_f32x2(v[e], slope_pair<TVB_ACT_SILU>(z[e]));
      break;
    default: break;
  }
}

}  // namespace tvb
