// What the tensor-core kernels of the fused linear layer share behind their accumulators: sixteen-bit loads and stores of a few
// neighbouring outputs, bias, activation, residual.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "linear_math.cuh"

namespace tvb {

// Two neighbouring 16-bit values as a pair of float32, and a pair rounded to two 16-bit values.
template <bool BF16>
__device__ __forceinline__ uint64_t unpack16(uint32_t w) {
  if (BF16) return ptx::pack_f32x2(w << 16, w & 0xffff0000u);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return ptx::pack_f32x2(__float_as_uint(f.x), __float_as_uint(f.y));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(uint64_t v) {
  float lo, hi;
  ptx::unpack_f32x2(v, lo, hi);
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool BF16>
__device__ __forceinline__ float load16(const void* p, int64_t i) {
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  return BF16 ? __uint_as_float(static_cast<uint32_t>(b) << 16) : __half2float(__ushort_as_half(b));
}

template <bool BF16>
__device__ __forceinline__ void store16(void* p, int64_t i, float v) {
  static_cast<uint16_t*>(p)[i] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// Up to 2 N values at element `at` (`count` of them exist), as pairs: one value at a time, for what does not begin on 16 bytes.
template <bool BF16, int N>
__device__ __forceinline__ void add_singly(const void* src, int64_t at, int count, uint64_t (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; e++) {
    const float a = 2 * e < count ? load16<BF16>(src, at + 2 * e) : 0.0f, b = 2 * e + 1 < count ? load16<BF16>(src, at + 2 * e + 1) : 0.0f;
    v[e] = ptx::add_f32x2(v[e], ptx::pack_f32x2(__float_as_uint(a), __float_as_uint(b)));
  }
}

template <bool BF16, int N>
__device__ __forceinline__ void store_singly(void* dst, int64_t at, int count, const uint64_t (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; e++) {
    float a, b;
    ptx::unpack_f32x2(v[e], a, b);
    if (2 * e < count) store16<BF16>(dst, at + 2 * e, a);
    if (2 * e + 1 < count) store16<BF16>(dst, at + 2 * e + 1, b);
  }
}

}  // namespace tvb
