// What the tensor-core kernels of the fused linear layer share behind their accumulators: sixteen-bit loads and stores of a few
// neighbouring outputs, bias, activation, residual.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "linear_math.cuh"

namespace tvb {

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
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
  static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(pack16<BF16>(v, v));
}

}  // namespace tvb
