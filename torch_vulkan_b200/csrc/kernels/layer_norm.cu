// Layer norm over the last dimension, forward and backward:
//   y = (x - mean) rstd g + b,   mean = <x>,   rstd = 1 / sqrt(<(x - mean)^2> + eps)        <.> the mean over a row
//   dx = rstd (u - <u> - h <u h>),   u = dy g,  h = (x - mean) rstd
//   dg = sum over rows of dy h,   db = sum over rows of dy
//
// Bound by memory: the forward pass reads and writes a row once, the backward pass reads two rows and writes one. All
// statistics and sums are float32; the variance is taken from the centred values, which a mean far from zero does not spoil.
//
// Forward: a group of T threads (8 or 32 of a warp, or a CTA) keeps its row in registers between the statistics and the result.
//
// Backward: persistent CTAs (512 threads per SM in all) stream their rows of x and dy through a ring in shared memory by bulk
// copies, so the next rows are on their way whatever the CTA does with the present ones, and keep the sums of dg and db of their
// columns in registers over all their rows. A cluster of two CTAs adds its sums through distributed shared memory and
// leaves one partial row in the workspace; a second kernel adds those in a fixed order (no atomics: the gradients repeat bit for
// bit). Rows that are short, or not whole 16-byte pieces, take the plain form of the kernel.
#include "../core/common.h"
#include "launch.h"
#include "numerics.cuh"
#include "ptx_pair.cuh"

namespace tvb {
namespace {

struct NormParams {
  const void* x;
  const void* dy;      // backward
  const void* weight;  // or NULL: 1
  const void* bias;    // or NULL: 0
  void* y;             // forward: y; backward: dx (or NULL)
  float* mean;
  float* rstd;
  float* partial;      // backward: [gridDim.x][2][d], or NULL
  int64_t x_ld, dy_ld, rows;
  int d, param_dtype;
  float eps;
};

// VEC values starting at element `i` (16 bytes when VEC > 1)
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* base, int64_t i, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = load_float<DT>(base, i);
  } else if constexpr (DT == TVB_F32) {
    const float4 t = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
    const uint4 t = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float2 f;
      if constexpr (DT == TVB_BF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
      else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}

// Two neighbouring 16-bit values as a pair of float32 (one register pair, for the instructions that work on both halves at once:
// with two bytes per value the kernels would be bound by their instructions, not by memory).
template <int DT>
__device__ __forceinline__ uint64_t pair16(uint32_t w) {
  if constexpr (DT == TVB_BF16) return ptx::pack_f32x2(w << 16, w & 0xffff0000u);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return ptx::pack_f32x2(__float_as_uint(f.x), __float_as_uint(f.y));
}

template <int DT>
__device__ __forceinline__ uint32_t round16(uint64_t v) {
  float lo, hi;
  ptx::unpack_f32x2(v, lo, hi);
  if constexpr (DT == TVB_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four neighbouring values as two pairs: 8 bytes of 16-bit values, 16 of float32.
template <int DT>
__device__ __forceinline__ void load_pairs(const void* base, int64_t i, uint64_t (&v)[2]) {
  if constexpr (DT == TVB_F32) {
    const uint4 t = *reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
    v[0] = ptx::pack_f32x2(t.x, t.y);
    v[1] = ptx::pack_f32x2(t.z, t.w);
  } else {
    const uint2 t = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
    v[0] = pair16<DT>(t.x);
    v[1] = pair16<DT>(t.y);
  }
}

template <int DT>
__device__ __forceinline__ void store_pairs(void* base, int64_t i, const uint64_t (&v)[2]) {
  if constexpr (DT == TVB_F32) {
    float a, b, c, d;
    ptx::unpack_f32x2(v[0], a, b);
    ptx::unpack_f32x2(v[1], c, d);
    *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(a, b, c, d);
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) = make_uint2(round16<DT>(v[0]), round16<DT>(v[1]));
  }
}

// 16 bytes of a row as pairs (VEC values), or one value.
template <int DT, int VEC>
struct Piece {
  static constexpr int kPairs = VEC / 2;
  uint64_t v[kPairs];
  __device__ __forceinline__ void load(const uint8_t* at) {
    if constexpr (DT == TVB_F32) {
      load_pairs<DT>(at, 0, v);
    } else {
      unpack(*reinterpret_cast<const uint4*>(at));
    }
  }
  __device__ __forceinline__ void unpack(const uint4& t) {
    v[0] = pair16<DT>(t.x); v[1] = pair16<DT>(t.y); v[2] = pair16<DT>(t.z); v[3] = pair16<DT>(t.w);
  }
  // weight or bias: of the values' type, or (WIDE) float32 beside 16-bit values
  template <bool WIDE>
  __device__ __forceinline__ void load_param(const uint8_t* at) {
    if constexpr (WIDE) {
#pragma unroll
      for (int e = 0; e < kPairs; e++) {
        const uint2 t = *reinterpret_cast<const uint2*>(at + 8 * e);
        v[e] = ptx::pack_f32x2(t.x, t.y);
      }
    } else {
      load(at);
    }
  }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int e = 0; e < kPairs; e++) v[e] = ptx::both_f32x2(f);
  }
  __device__ __forceinline__ void store(uint8_t* at) const {
    if constexpr (DT == TVB_F32) store_pairs<DT>(at, 0, v);
    else *reinterpret_cast<uint4*>(at) = make_uint4(round16<DT>(v[0]), round16<DT>(v[1]), round16<DT>(v[2]), round16<DT>(v[3]));
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < kPairs; e++) v[e] = 0;
  }
  __device__ __forceinline__ float sum() const {
    uint64_t s = v[0];
#pragma unroll
    for (int e = 1; e < kPairs; e++) s = ptx::add_f32x2(s, v[e]);
    return ptx::sum_f32x2(s);
  }
  // subtracts the mean; returns the sum of the squares
  __device__ __forceinline__ float center(float mean) {
    const uint64_t m = ptx::both_f32x2(-mean);
    uint64_t s = 0;
#pragma unroll
    for (int e = 0; e < kPairs; e++) {
      v[e] = ptx::add_f32x2(v[e], m);
      s = ptx::fma_f32x2(v[e], v[e], s);
    }
    return ptx::sum_f32x2(s);
  }
  __device__ __forceinline__ void scale(float rstd, const Piece& g, const Piece& b) {
    const uint64_t r = ptx::both_f32x2(rstd);
#pragma unroll
    for (int e = 0; e < kPairs; e++) v[e] = ptx::fma_f32x2(ptx::mul_f32x2(v[e], r), g.v[e], b.v[e]);
  }
};
template <int DT>
struct Piece<DT, 1> {
  float v;
  __device__ __forceinline__ void load(const uint8_t* at) { v = load_float<DT>(at, 0); }
  template <bool WIDE>
  __device__ __forceinline__ void load_param(const uint8_t* at) {
    v = WIDE ? *reinterpret_cast<const float*>(at) : load_float<DT>(at, 0);
  }
  __device__ __forceinline__ void fill(float f) { v = f; }
  __device__ __forceinline__ void store(uint8_t* at) const { store_float<DT>(at, 0, v); }
  __device__ __forceinline__ void zero() { v = 0.0f; }
  __device__ __forceinline__ float sum() const { return v; }
  __device__ __forceinline__ float center(float mean) {
    v -= mean;
    return v * v;
  }
  __device__ __forceinline__ void scale(float rstd, const Piece& g, const Piece& b) { v = fmaf(v * rstd, g.v, b.v); }
};

template <int DT, int VEC>
__device__ __forceinline__ void store_vec(void* base, int64_t i, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    store_float<DT>(base, i, v[0]);
  } else if constexpr (DT == TVB_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (DT == TVB_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The parameters are of x's type or float32.
template <int DT, int VEC>
__device__ __forceinline__ void load_param(const void* base, int param_dtype, int i, float other, float (&v)[VEC]) {
  if (base == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = other;
  } else if (DT == TVB_F32 || param_dtype != TVB_F32) {
    load_vec<DT, VEC>(base, i, v);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = static_cast<const float*>(base)[i + j];
  }
}

// Two values summed over a warp: the first exchange leaves each half of the lanes one of them (five shuffles instead of ten).
// Lanes 0-15 get the sum of a, lanes 16-31 that of b.
__device__ __forceinline__ float fold2(float a, float b) {
  const bool up = (threadIdx.x & 16) != 0;
  float s = up ? b : a;
  s += __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
  for (int x = 8; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  return s;
}

// The same over a CTA of `warps` warps, every thread getting both. buf: room for `warps` pairs, another one at every second
// call (a thread may still be reading one when the next call begins).
__device__ __forceinline__ void cta_sum2(float& a, float& b, float2* buf, int warps) {
  const int lane = threadIdx.x & 31;
  float s = fold2(a, b);
  if ((lane & 15) == 0) reinterpret_cast<float*>(buf + (threadIdx.x >> 5))[lane >> 4] = s;
  __syncthreads();
  const float2 v = lane < warps ? buf[lane] : make_float2(0.0f, 0.0f);
  s = fold2(v.x, v.y);
  a = __shfl_sync(0xffffffffu, s, 0);
  b = __shfl_sync(0xffffffffu, s, 16);
}

// Sums of N (one or two) values over the T threads of a group (a power of two up to a warp, or the whole CTA); every thread gets
// them.
template <int T, int N = 2>
__device__ __forceinline__ void group_sum(float& a, float& b, float2 (*buf)[32], int slot) {
  if constexpr (T > 32 && N == 2) {
    cta_sum2(a, b, buf[slot], T / 32);
  } else {
#pragma unroll
    for (int s = (T < 32 ? T : 32) / 2; s > 0; s >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, s);
      if constexpr (N == 2) b += __shfl_xor_sync(0xffffffffu, b, s);
    }
    if constexpr (T > 32) {
      float* one = reinterpret_cast<float*>(buf[slot]);
      if ((threadIdx.x & 31) == 0) one[threadIdx.x >> 5] = a;
      __syncthreads();
      a = 0.0f;
      if constexpr (T <= 256) {
#pragma unroll
        for (int w = 0; w < T / 32; w++) a += one[w];
      } else {
        a = (threadIdx.x & 31) < T / 32 ? one[threadIdx.x & 31] : 0.0f;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) a += __shfl_xor_sync(0xffffffffu, a, s);
      }
    }
  }
}

template <int T>
constexpr int norm_threads() { return T < 128 ? 128 : T; }

constexpr int kRingStages = 8;  // rows on their way in the forward kernel, at most
constexpr int kValsBwd = 16;   // values of a row per thread in the backward kernels (with two sums per value)

// At least this many CTAs per SM: 1024 threads of 64 registers, but for 16-bit rows of up to 4096 values, where a few registers
// more are worth more than the threads.
template <int VEC, int T>
constexpr int norm_ctas_per_sm() { return VEC == 8 && T < 512 ? 1 : 1024 / norm_threads<T>(); }

// The weight's and bias's part of a row's result, with parameters of one width: x = (x rstd) g + b, stored.
template <int DT, int VEC, int T, int VALS, int ROWS, bool WIDE>
__device__ __forceinline__ void norm_finish(const NormParams& p, Piece<DT, VEC> (&x)[ROWS][VALS / VEC], const float (&rstd)[ROWS],
                                            const bool (&live)[ROWS], int64_t row, int t) {
  constexpr int kSize = DT == TVB_F32 ? 4 : 2, kWidth = WIDE ? 4 : kSize, kPieces = VALS / VEC;
  const uint8_t* g_at = static_cast<const uint8_t*>(p.weight) + t * VEC * kWidth;
  const uint8_t* b_at = static_cast<const uint8_t*>(p.bias) + t * VEC * kWidth;
  uint8_t* y_at[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; k++) y_at[k] = static_cast<uint8_t*>(p.y) + ((row + k) * p.d + t * VEC) * kSize;
#pragma unroll
  for (int c = 0; c < kPieces; c++) {
    if ((c * T + t) * VEC >= p.d) continue;
    Piece<DT, VEC> g, b;
    if (p.weight != nullptr) g.template load_param<WIDE>(g_at + c * T * VEC * kWidth);
    else g.fill(1.0f);
    if (p.bias != nullptr) b.template load_param<WIDE>(b_at + c * T * VEC * kWidth);
    else b.fill(0.0f);
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      x[k][c].scale(rstd[k], g, b);
      if (live[k]) x[k][c].store(y_at[k] + c * T * VEC * kSize);
    }
  }
}

// VALS values of each of ROWS rows per thread: two rows share the loads and conversions of the parameters and the barriers.
template <int DT, int VEC, int T, int VALS, int ROWS>
__global__ void __launch_bounds__(norm_threads<T>(), norm_ctas_per_sm<VEC, T>()) layer_norm_kernel(const NormParams p) {
  constexpr int kGroups = norm_threads<T>() / T, kPieces = VALS / VEC, kSize = DT == TVB_F32 ? 4 : 2;
  __shared__ float2 buf[2][32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int t = threadIdx.x % T;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / T) * ROWS;
  Piece<DT, VEC> x[ROWS][kPieces];
  float sum[2] = {}, sq[2] = {}, mean[ROWS], rstd[ROWS];
  bool live[ROWS];  // (every thread takes part in the sums)
#pragma unroll
  for (int k = 0; k < ROWS; k++) {
    live[k] = row + k < p.rows;
    const uint8_t* at = static_cast<const uint8_t*>(p.x) + ((row + k) * p.x_ld + t * VEC) * kSize;
#pragma unroll
    for (int c = 0; c < kPieces; c++) {
      if (live[k] && (c * T + t) * VEC < p.d) x[k][c].load(at + c * T * VEC * kSize);
      else x[k][c].zero();
    }
  }
#pragma unroll
  for (int k = 0; k < ROWS; k++)
#pragma unroll
    for (int c = 0; c < kPieces; c++) sum[k] += x[k][c].sum();
  group_sum<T, ROWS>(sum[0], sum[1], buf, 0);
#pragma unroll
  for (int k = 0; k < ROWS; k++) {
    mean[k] = sum[k] / static_cast<float>(p.d);
#pragma unroll
    for (int c = 0; c < kPieces; c++)
      if ((c * T + t) * VEC < p.d) sq[k] += x[k][c].center(mean[k]);
  }
  group_sum<T, ROWS>(sq[0], sq[1], buf, 1);
#pragma unroll
  for (int k = 0; k < ROWS; k++) {
    rstd[k] = 1.0f / sqrtf(sq[k] / static_cast<float>(p.d) + p.eps);
    if (t == 0 && live[k]) {
      if (p.mean != nullptr) p.mean[row + k] = mean[k];
      if (p.rstd != nullptr) p.rstd[row + k] = rstd[k];
    }
  }
  if (DT != TVB_F32 && p.param_dtype == TVB_F32) norm_finish<DT, VEC, T, VALS, ROWS, true>(p, x, rstd, live, row, t);
  else norm_finish<DT, VEC, T, VALS, ROWS, false>(p, x, rstd, live, row, t);
}

// Rows too long for the registers of a CTA: three passes over the row (the second and third mostly from the L2).
template <int DT>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(const NormParams p) {
  __shared__ float2 buf[2][32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int64_t row = blockIdx.x, base = row * p.x_ld;
  float sum = 0.0f, sq = 0.0f, none = 0.0f;
  for (int c = threadIdx.x; c < p.d; c += 1024) sum += load_float<DT>(p.x, base + c);
  group_sum<1024>(sum, none, buf, 0);
  const float mean = sum / static_cast<float>(p.d);
  for (int c = threadIdx.x; c < p.d; c += 1024) {
    const float v = load_float<DT>(p.x, base + c) - mean;
    sq = fmaf(v, v, sq);
  }
  group_sum<1024>(sq, none, buf, 1);
  const float rstd = 1.0f / sqrtf(sq / static_cast<float>(p.d) + p.eps);
  if (threadIdx.x == 0) {
    if (p.mean != nullptr) p.mean[row] = mean;
    if (p.rstd != nullptr) p.rstd[row] = rstd;
  }
  for (int c = threadIdx.x; c < p.d; c += 1024) {
    float g[1], b[1];
    load_param<DT, 1>(p.weight, p.param_dtype, c, 1.0f, g);
    load_param<DT, 1>(p.bias, p.param_dtype, c, 0.0f, b);
    store_float<DT>(p.y, row * p.d + c, fmaf((load_float<DT>(p.x, base + c) - mean) * rstd, g[0], b[0]));
  }
}

template <int DT, int VEC, int T>
__global__ void __launch_bounds__(norm_threads<T>()) layer_norm_backward_kernel(const NormParams p) {
  constexpr int kChunks = kValsBwd / VEC, kGroups = norm_threads<T>() / T;
  __shared__ float2 buf[2][32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int t = threadIdx.x % T;
  float dg[kChunks][VEC] = {}, db[kChunks][VEC] = {};
  const float inv_d = 1.0f / static_cast<float>(p.d);
  int slot = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups; row0 < p.rows; row0 += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = row0 + threadIdx.x / T;
    const bool live = row < p.rows;
    const float mean = live ? p.mean[row] : 0.0f, rstd = live ? p.rstd[row] : 0.0f;
    float h[kChunks][VEC], u[kChunks][VEC];
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int col = (c * T + t) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; j++) h[c][j] = u[c][j] = 0.0f;
      if (live && col < p.d) {
        load_vec<DT, VEC>(p.x, row * p.x_ld + col, h[c]);
        load_vec<DT, VEC>(p.dy, row * p.dy_ld + col, u[c]);
      }
    }
    float su = 0.0f, suh = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int col = (c * T + t) * VEC;
      if (!live || col >= p.d) continue;
      float g[VEC];
      load_param<DT, VEC>(p.weight, p.param_dtype, col, 1.0f, g);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        h[c][j] = (h[c][j] - mean) * rstd;
        dg[c][j] = fmaf(u[c][j], h[c][j], dg[c][j]);
        db[c][j] += u[c][j];
        u[c][j] *= g[j];
        su += u[c][j];
        suh = fmaf(u[c][j], h[c][j], suh);
      }
    }
    if (p.y == nullptr) continue;
    group_sum<T>(su, suh, buf, slot);
    slot ^= 1;
    const float mu = su * inv_d, muh = suh * inv_d;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int col = (c * T + t) * VEC;
      if (!live || col >= p.d) continue;
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) o[j] = rstd * (u[c][j] - mu - h[c][j] * muh);
      store_vec<DT, VEC>(p.y, row * p.d + col, o);
    }
  }
  if (p.partial == nullptr) return;
  if constexpr (kGroups > 1) {
    // the CTA's groups hold the same columns: their sums are added through shared memory, group 0 first
    __shared__ float fold[kGroups][T * kValsBwd + 1];
    float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.d;
#pragma unroll
    for (int which = 0; which < 2; which++) {
#pragma unroll
      for (int c = 0; c < kChunks; c++)
#pragma unroll
        for (int j = 0; j < VEC; j++) fold[threadIdx.x / T][(c * T + t) * VEC + j] = which == 0 ? dg[c][j] : db[c][j];
      __syncthreads();
      for (int col = threadIdx.x; col < p.d; col += norm_threads<T>()) {
        float s = 0.0f;
#pragma unroll
        for (int g = 0; g < kGroups; g++) s += fold[g][col];
        out[which * p.d + col] = s;
      }
      __syncthreads();
    }
  } else {
    float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.d;
#pragma unroll
    for (int c = 0; c < kChunks; c++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const int col = (c * T + t) * VEC + j;
        if (col < p.d) {
          out[col] = dg[c][j];
          out[p.d + col] = db[c][j];
        }
      }
  }
}

// Bytes from global memory into this CTA's shared memory (both on 16 bytes, a multiple of 16), counted at `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}

// Forward, long rows of 16-bit values: persistent CTAs, one per SM, whose rows come through a ring in shared memory by bulk
// copies, so the next ones are on their way during a row's sums and barriers. 32 values of a row per thread; the parameters stay
// in registers, as they are. (bfloat16, us, with registers and 1024 threads per row before: 4096 x 16384 71 -> 56, 8192 x 12288
// 119 -> 87, 300 x 16384 8.9 -> 7.0. Up to 8192 values two CTAs' rows hide each other's barriers as well without a ring.)
template <int DT, int T>
__global__ void __launch_bounds__(T, 1) layer_norm_ring_kernel(const NormParams p, const int stages, int* status) {
  constexpr int kPieces = 4;
  using Values = Piece<DT, 8>;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float2 buf[2][32];
  __shared__ uint64_t bars[kRingStages];
  __shared__ int abort_flag;
  const int d = p.d, row_bytes = d * 2, t = threadIdx.x;
  const int left = d - 8 * t;  // piece c of this thread (columns 8 (c T + t) ...) exists if left > 8 c T
  const uint32_t ring0 = ptx::smem_u32(ring), bar0 = ptx::smem_u32(bars);
  if (t == 0) {
    for (int s = 0; s < stages; s++) ptx::mbar_init(bar0 + 8 * s, 1);
    abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int64_t step = gridDim.x;
  const int count = blockIdx.x < p.rows ? static_cast<int>((p.rows - blockIdx.x + step - 1) / step) : 0;
  const uint8_t* next = static_cast<const uint8_t*>(p.x) + blockIdx.x * p.x_ld * 2;  // the next row to fetch (thread 0)
  int fetched = 0;
  auto fetch = [&](int slot) {
    ptx::mbar_expect_tx(bar0 + 8 * slot, row_bytes);
    bulk_load(ring0 + slot * row_bytes, next, row_bytes, bar0 + 8 * slot);
    next += step * p.x_ld * 2;
    fetched++;
  };
  if (t == 0)
    while (fetched < count && fetched < stages) fetch(fetched);
  const uint32_t one = DT == TVB_BF16 ? 0x3f803f80u : 0x3c003c00u;
  uint4 g[kPieces], b[kPieces];
#pragma unroll
  for (int c = 0; c < kPieces; c++) {
    g[c] = make_uint4(one, one, one, one);
    b[c] = make_uint4(0, 0, 0, 0);
    if (left <= 8 * c * T) continue;
    if (p.weight != nullptr) g[c] = static_cast<const uint4*>(p.weight)[c * T + t];
    if (p.bias != nullptr) b[c] = static_cast<const uint4*>(p.bias)[c * T + t];
  }
  int slot = 0, before = 0;
  uint32_t phase = 0;
  int64_t row = blockIdx.x;
#pragma unroll 1
  for (int i = 0; i < count; i++, row += step) {
    ptx::mbar_wait(bar0 + 8 * slot, phase, &abort_flag);  // (no early exit: barriers follow)
    const uint8_t* mine = ring + static_cast<size_t>(slot) * row_bytes + t * 16;
    Values x[kPieces];
    float sum = 0.0f, sq = 0.0f, none = 0.0f;
#pragma unroll
    for (int c = 0; c < kPieces; c++) {
      x[c].zero();
      if (left > 8 * c * T) x[c].load(mine + c * T * 16);
      sum += x[c].sum();
    }
    group_sum<T, 1>(sum, none, buf, 0);
    if (t == 0 && i >= 1 && fetched < count) fetch(before);  // (all threads have read the row before)
    const float mean = sum / static_cast<float>(d);
#pragma unroll
    for (int c = 0; c < kPieces; c++)
      if (left > 8 * c * T) sq += x[c].center(mean);
    group_sum<T, 1>(sq, none, buf, 1);
    const float rstd = 1.0f / sqrtf(sq / static_cast<float>(d) + p.eps);
    if (t == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
    uint8_t* y = static_cast<uint8_t*>(p.y) + row * row_bytes + t * 16;
#pragma unroll
    for (int c = 0; c < kPieces; c++) {
      if (left <= 8 * c * T) continue;
      Values gv, bv;
      gv.unpack(g[c]);
      bv.unpack(b[c]);
      x[c].scale(rstd, gv, bv);
      x[c].store(y + c * T * 16);
    }
    before = slot;
    if (++slot == stages) {
      slot = 0;
      phase ^= 1u;
    }
  }
  __syncthreads();
  if (t == 0 && abort_flag != 0) atomicExch(status, 2);
}

constexpr int kRingCluster = 2;

// The streamed form: `stages` slots of one row of x and one of dy each. Row number i of this CTA (row blockIdx.x + i *
// gridDim.x) lies in slot i % stages; the slot of row i - 1 is refilled behind the barrier inside row i's sums, which every thread
// reaches only after it is done with row i - 1. A row is read from shared memory twice (for the sums, for dx), which leaves the
// registers to the column sums and, where they are 16-bit, the weights; others (WIDE: float32) lie in shared memory.
// 8192 x 8192 bfloat16: 84 us, 4.8 TB/s, with 53 % of the issue slots used: neither memory nor instructions are at their limit; what is
// left is the block-wide sum per row, which one CTA per SM cannot hide behind another's. (The instructions were twice as many
// with the number of threads a variable, most of them addresses.)
// Dynamic shared memory: the ring, the weights (WIDE), two buffers for the sums over the warps.
template <int DT, int T, int UNITS, bool WIDE>
__global__ void __launch_bounds__(T, 512 / T) layer_norm_backward_ring_kernel(const NormParams p, const int stages, int* status) {
  constexpr int kSize = DT == TVB_F32 ? 4 : 2, kUnits = UNITS, threads = T, warps = T / 32;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t bars[8];
  __shared__ int abort_flag;
  const int d = p.d, row_bytes = d * kSize, t = threadIdx.x;
  const int left = d - 4 * t;  // unit c of this thread (columns 4 (c T + t) ...) exists if left > 4 c T
  float* weights = reinterpret_cast<float*>(ring + static_cast<size_t>(stages) * 2 * row_bytes);
  float2* buf = reinterpret_cast<float2*>(weights + (WIDE ? d : 0));
  const uint32_t ring0 = ptx::smem_u32(ring), bar0 = ptx::smem_u32(bars);
  if (t == 0) {
    for (int s = 0; s < stages; s++) ptx::mbar_init(bar0 + 8 * s, 1);
    abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int64_t step = gridDim.x;
  const int count = blockIdx.x < p.rows ? static_cast<int>((p.rows - blockIdx.x + step - 1) / step) : 0;
  const uint8_t* next_x = static_cast<const uint8_t*>(p.x) + blockIdx.x * p.x_ld * kSize;  // the next row to fetch (thread 0)
  const uint8_t* next_dy = static_cast<const uint8_t*>(p.dy) + blockIdx.x * p.dy_ld * kSize;
  int fetched = 0;
  auto fetch = [&](int slot) {
    const uint32_t dst = ring0 + 2 * slot * row_bytes, bar = bar0 + 8 * slot;
    ptx::mbar_expect_tx(bar, 2 * row_bytes);
    bulk_load(dst, next_x, row_bytes, bar);
    bulk_load(dst + row_bytes, next_dy, row_bytes, bar);
    next_x += step * p.x_ld * kSize;
    next_dy += step * p.dy_ld * kSize;
    fetched++;
  };
  if (t == 0)
    while (fetched < count && fetched < stages) fetch(fetched);
  uint64_t dg[kUnits][2] = {}, db[kUnits][2] = {};
  uint2 kept[kUnits];  // !WIDE: the weights as they are
#pragma unroll
  for (int c = 0; c < kUnits; c++) {
    kept[c] = make_uint2(0, 0);
    if (left <= 4 * c * T) continue;
    const int col = 4 * (c * T + t);
    if constexpr (WIDE) {  // (every thread reads back only what it wrote)
      *reinterpret_cast<float4*>(weights + col) = p.weight != nullptr ? *reinterpret_cast<const float4*>(static_cast<const float*>(p.weight) + col)
                                                                      : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    } else {
      const uint32_t one = DT == TVB_BF16 ? 0x3f803f80u : 0x3c003c00u;
      kept[c] = p.weight != nullptr ? *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.weight) + col) : make_uint2(one, one);
    }
  }
  auto weight = [&](int c, uint64_t (&g)[2]) {
    if constexpr (WIDE) {
      load_pairs<TVB_F32>(weights, 4 * (c * T + t), g);
    } else {
      g[0] = pair16<DT>(kept[c].x);
      g[1] = pair16<DT>(kept[c].y);
    }
  };
  const float inv_d = 1.0f / static_cast<float>(d);
  const float* mean_at = p.mean + blockIdx.x;
  const float* rstd_at = p.rstd + blockIdx.x;
  uint8_t* y_at = p.y == nullptr ? nullptr : static_cast<uint8_t*>(p.y) + static_cast<int64_t>(blockIdx.x) * row_bytes + t * 4 * kSize;
  const int64_t y_step = step * row_bytes;
  float mean = count > 0 ? *mean_at : 0.0f, rstd = count > 0 ? *rstd_at : 0.0f;
  int slot = 0, before = 0;
  uint32_t phase = 0;
  const uint8_t* mine = ring + t * 4 * kSize;  // this thread's first unit of the row of x in the present slot
#pragma unroll 1
  for (int i = 0; i < count; i++) {
    float next_mean = 0.0f, next_rstd = 0.0f;  // the next row's statistics are asked for a row ahead
    mean_at += step;
    rstd_at += step;
    if (i + 1 < count) {
      next_mean = *mean_at;
      next_rstd = *rstd_at;
    }
    ptx::mbar_wait(bar0 + 8 * slot, phase, &abort_flag);  // (no early exit: barriers follow)
    const uint8_t* xs = mine;
    const uint8_t* ds = mine + row_bytes;
    const uint64_t m2 = ptx::both_f32x2(-mean), r2 = ptx::both_f32x2(rstd);
    uint64_t su2 = 0, sux2 = 0;
#pragma unroll
    for (int c = 0; c < kUnits; c++) {
      if (left <= 4 * c * T) continue;
      uint64_t x[2], dy[2], g[2];
      load_pairs<DT>(xs, 4 * c * T, x);
      load_pairs<DT>(ds, 4 * c * T, dy);
      weight(c, g);
#pragma unroll
      for (int e = 0; e < 2; e++) {
        x[e] = ptx::add_f32x2(x[e], m2);
        db[c][e] = ptx::add_f32x2(db[c][e], dy[e]);
        dg[c][e] = ptx::fma_f32x2(ptx::mul_f32x2(x[e], r2), dy[e], dg[c][e]);
        const uint64_t u = ptx::mul_f32x2(dy[e], g[e]);
        su2 = ptx::add_f32x2(su2, u);
        sux2 = ptx::fma_f32x2(u, x[e], sux2);
      }
    }
    float su = ptx::sum_f32x2(su2), sux = ptx::sum_f32x2(sux2);
    cta_sum2(su, sux, buf + (i & 1) * warps, warps);
    if (t == 0 && i >= 1 && fetched < count) fetch(before);
    if (y_at != nullptr) {
      // dx = rstd u - rstd <u> - (x - mean) rstd^2 <u h>,  <u h> = rstd <u (x - mean)>
      const uint64_t c0 = ptx::both_f32x2(-su * inv_d * rstd), c1 = ptx::both_f32x2(-(rstd * (rstd * sux * inv_d)) * rstd);
#pragma unroll
      for (int c = 0; c < kUnits; c++) {
        if (left <= 4 * c * T) continue;
        uint64_t x[2], dy[2], g[2];
        load_pairs<DT>(xs, 4 * c * T, x);
        load_pairs<DT>(ds, 4 * c * T, dy);
        weight(c, g);
#pragma unroll
        for (int e = 0; e < 2; e++)
          x[e] = ptx::fma_f32x2(ptx::add_f32x2(x[e], m2), c1, ptx::fma_f32x2(dy[e], ptx::mul_f32x2(g[e], r2), c0));
        store_pairs<DT>(y_at, 4 * c * T, x);
      }
      y_at += y_step;
    }
    mean = next_mean;
    rstd = next_rstd;
    before = slot;
    mine += 2 * row_bytes;
    if (++slot == stages) {
      slot = 0;
      phase ^= 1u;
      mine = ring + t * 4 * kSize;
    }
  }
  __syncthreads();
  if (t == 0 && abort_flag != 0) atomicExch(status, 2);
  if (p.partial == nullptr) return;
  // the cluster's sums: each CTA leaves its own in shared memory (the ring is idle), and adds up half of the columns
  float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int c = 0; c < kUnits; c++) {
    if (left <= 4 * c * T) continue;
    const int col = 4 * (c * T + t);
    store_pairs<TVB_F32>(sums, col, dg[c]);
    store_pairs<TVB_F32>(sums, d + col, db[c]);
  }
  ptx::cluster_sync();
  const uint32_t rank = ptx::cluster_ctarank();
  float* out = p.partial + static_cast<int64_t>(blockIdx.x / kRingCluster) * 2 * p.d;
  const int share = 2 * p.d / kRingCluster;
  for (int e = t; e < share; e += threads) {
    const int at = static_cast<int>(rank) * share + e;
    float v = 0.0f;
#pragma unroll
    for (uint32_t r = 0; r < kRingCluster; r++) {
      float w;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(ptx::mapa(ring0 + 4 * at, r)) : "memory");
      v += w;
    }
    out[at] = v;
  }
  ptx::cluster_sync();  // no CTA's shared memory is released while another may read it
}

// Rows too long for the registers: dx in two passes over the row; the sums over the rows in a kernel of their own.
template <int DT>
__global__ void __launch_bounds__(1024) layer_norm_backward_long_kernel(const NormParams p) {
  __shared__ float2 buf[2][32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int64_t row = blockIdx.x;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float su = 0.0f, suh = 0.0f;
  for (int pass = 0; pass < 2; pass++) {
    for (int c = threadIdx.x; c < p.d; c += 1024) {
      float g[1];
      load_param<DT, 1>(p.weight, p.param_dtype, c, 1.0f, g);
      const float h = (load_float<DT>(p.x, row * p.x_ld + c) - mean) * rstd, u = load_float<DT>(p.dy, row * p.dy_ld + c) * g[0];
      if (pass == 0) {
        su += u;
        suh = fmaf(u, h, suh);
      } else {
        store_float<DT>(p.y, row * p.d + c, rstd * (u - su - h * suh));
      }
    }
    if (pass == 0) {
      group_sum<1024>(su, suh, buf, 0);
      su /= static_cast<float>(p.d);
      suh /= static_cast<float>(p.d);
    }
  }
}

// (for rows too long for the registers) one CTA row of the grid per slice of the rows, 256 columns per CTA
template <int DT>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const NormParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int col = static_cast<int>(blockIdx.x) * 256 + threadIdx.x;
  if (col >= p.d) return;
  const int64_t begin = p.rows * blockIdx.y / gridDim.y, end = p.rows * (blockIdx.y + 1) / gridDim.y;
  float dg = 0.0f, db = 0.0f;
  for (int64_t row = begin; row < end; row++) {
    const float dy = load_float<DT>(p.dy, row * p.dy_ld + col);
    dg = fmaf(dy, (load_float<DT>(p.x, row * p.x_ld + col) - p.mean[row]) * p.rstd[row], dg);
    db += dy;
  }
  float* out = p.partial + static_cast<int64_t>(blockIdx.y) * 2 * p.d;
  out[col] = dg;
  out[p.d + col] = db;
}

// The partial rows added up: 32 columns per CTA, eight threads per column taking every eighth row, in a fixed order.
__global__ void __launch_bounds__(256) layer_norm_reduce_kernel(const float* partial, int parts, int d, void* dweight, void* dbias,
                                                                int param_dtype) {
  __shared__ float fold[8][33];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int col = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.0f;
  if (col < 2 * d)
    for (int r = g; r < parts; r += 8) s += partial[static_cast<int64_t>(r) * 2 * d + col];
  fold[g][lane] = s;
  __syncthreads();
  if (g != 0 || col >= 2 * d) return;
  s = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; r++) s += fold[r][lane];
  void* out = col < d ? dweight : dbias;
  if (out != nullptr) store_float_rt(out, col < d ? col : col - d, param_dtype, s);
}

constexpr int kRingRoom = 224 * 1024;       // shared memory of the forward kernel's ring, at most
constexpr int kLongest = 32 * 1024;         // values of a row that the forward kernels keep in registers
constexpr int kLongestBwd = 16 * 1024;      // and the plain backward kernel
constexpr int64_t kLongSlices = 64;         // partial rows of layer_norm_columns_kernel, at most

int norm_group(int64_t d, int vals) {
  for (int t : {8, 32, 128, 256, 512})
    if (d <= static_cast<int64_t>(t) * vals) return t;
  return 1024;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The streamed backward kernel: rows of 512 to 16384 values that fit the shared memory at least twice. (A few numbers of threads, so that they can be constants of the
// kernel.) A thread owns 16 columns, or 32 beyond 8192: 512 threads of up to 128 registers per SM (1024 of 64 spilled, 108 us against
// 84 at 8192 x 8192 bfloat16; 32 columns for all: 85, but 152 against 144 at 16384 x 4096 float32).
struct Ring {
  int cols, threads, per_sm, stages;
  size_t smem;
};
Ring ring_shape(int64_t d, int es, bool wide) {
  Ring r{};
  if (d < 512 || d > 16384 || d % 4 != 0) return r;
  r.cols = d <= 8192 ? 16 : 32;
  for (int t : {64, 128, 192, 256, 384, 512})
    if (r.threads == 0 && d <= t * r.cols) r.threads = t;
  r.per_sm = 512 / r.threads;
  const int64_t rest = (wide ? d * 4 : 0) + r.threads / 2;  // weights, sums over the warps
  // (228 KB per SM, of which every CTA takes 1 KB for itself and some for its barriers)
  r.stages = static_cast<int>(std::min<int64_t>((228 * 1024 / r.per_sm - 1024 - 128 - rest) / (2 * d * es), 8));
  if (r.stages < 2) return Ring{};
  r.smem = static_cast<size_t>(std::max<int64_t>(r.stages * 2 * d * es + rest, 8 * d));  // (the sums of 2 d columns at the end)
  return r;
}

// Its CTAs: whole clusters, at most what the GPU holds, no more than there are rows.
int64_t ring_ctas(int64_t rows, const Ring& r) { return std::min(ceil_div(rows, kRingCluster) * kRingCluster, static_cast<int64_t>(148) * r.per_sm); }

// CTAs of the plain backward kernel (and partial rows of its sums).
int64_t norm_parts(int64_t rows, int64_t d) {
  if (d > kLongestBwd) return std::min<int64_t>(rows, kLongSlices);
  const int t = norm_group(d, kValsBwd);
  const int64_t groups = t < 128 ? 128 / t : 1;
  const int64_t most = t <= 128 ? 148 * 4 : (t == 256 ? 148 * 2 : 148);
  return std::min(ceil_div(rows, groups), most);
}

// The forward kernel's shape: as few threads as hold a row (bfloat16, us: 65536 x 768 with a warp per row 42, a CTA of 128 for two
// rows 76; 65536 x 512 with 32 values of one row per thread 35, 16 of two rows 28; 16384 x 4096 50 and 56; 16384 x 5120 with 384
// threads 84, with 512 94).
template <int DT, int VEC>
int forward_vec(cudaStream_t stream, const NormParams& p) {
  auto run = [&](auto kernel, int t, int rows) {
    const int64_t per_cta = (t < 128 ? 128 / t : 1) * rows;
    return launch_dependent("layer_norm", kernel, dim3(static_cast<unsigned>(ceil_div(p.rows, per_cta))), dim3(t < 128 ? 128 : t), 0, stream, p);
  };
  if (p.d <= 16 * 8) return run(layer_norm_kernel<DT, VEC, 8, 16, 2>, 8, 2);
  if (p.d <= 32 * 8) return run(layer_norm_kernel<DT, VEC, 8, 32, 1>, 8, 1);
  if (p.d <= 16 * 32) return run(layer_norm_kernel<DT, VEC, 32, 16, 2>, 32, 2);
  if (p.d <= 32 * 32) return run(layer_norm_kernel<DT, VEC, 32, 32, 1>, 32, 1);
  if (p.d <= 16 * 128) return run(layer_norm_kernel<DT, VEC, 128, 16, 2>, 128, 2);
  if (p.d <= 32 * 128) return run(layer_norm_kernel<DT, VEC, 128, 32, 1>, 128, 1);
  if (p.d <= 16 * 384) return run(layer_norm_kernel<DT, VEC, 384, 16, 2>, 384, 2);
  if (p.d <= 16 * 512) return run(layer_norm_kernel<DT, VEC, 512, 16, 2>, 512, 2);
  if (p.d <= 16 * 1024) return run(layer_norm_kernel<DT, VEC, 1024, 16, 2>, 1024, 2);
  return run(layer_norm_kernel<DT, VEC, 1024, 32, 1>, 1024, 1);
}

template <int DT, int VEC>
int backward_vec(cudaStream_t stream, const NormParams& p, int64_t parts) {
  const int t = norm_group(p.d, kValsBwd);
  auto kernel = t == 8 ? layer_norm_backward_kernel<DT, VEC, 8> : layer_norm_backward_kernel<DT, VEC, 32>;
  if constexpr (VEC == 1) {
    if (t >= 128)
      kernel = t == 128 ? layer_norm_backward_kernel<DT, VEC, 128> : t == 256 ? layer_norm_backward_kernel<DT, VEC, 256>
             : t == 512 ? layer_norm_backward_kernel<DT, VEC, 512> : layer_norm_backward_kernel<DT, VEC, 1024>;
  } else {  // (the rest goes through the ring, but for float32 rows of which it cannot hold two)
    if (t > 32) {
      if constexpr (DT != TVB_F32) return fail("tvb_layer_norm_backward: no kernel for this row");
      else kernel = layer_norm_backward_kernel<DT, VEC, 1024>;
    }
  }
  return launch_dependent("layer_norm_backward", kernel, dim3(static_cast<unsigned>(parts)), dim3(t < 128 ? 128 : t), 0, stream, p);
}

template <int DT, int T, int UNITS, bool WIDE>
int backward_ring(int device, cudaStream_t stream, const NormParams& p, const Ring& r, int64_t ctas) {
  auto kernel = layer_norm_backward_ring_kernel<DT, T, UNITS, WIDE>;
  static bool configured[64] = {};
  if (!configured[device & 63]) {
    TVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 128));
    configured[device & 63] = true;
  }
  int* status = nullptr;
  if (status_word(device, &status) != 0) return -1;
  return launch_dependent_cluster("layer_norm_backward_ring", kernel, kRingCluster, dim3(static_cast<unsigned>(ctas)), dim3(T), r.smem, stream, p,
                                  r.stages, status);
}

template <int DT, bool WIDE>
int backward_ring_threads(int device, cudaStream_t stream, const NormParams& p, const Ring& r, int64_t ctas) {
  if (r.cols == 32) {
    if (r.threads == 384) return backward_ring<DT, 384, 8, WIDE>(device, stream, p, r, ctas);
    return backward_ring<DT, 512, 8, WIDE>(device, stream, p, r, ctas);
  }
  switch (r.threads) {
    case 64: return backward_ring<DT, 64, 4, WIDE>(device, stream, p, r, ctas);
    case 128: return backward_ring<DT, 128, 4, WIDE>(device, stream, p, r, ctas);
    case 192: return backward_ring<DT, 192, 4, WIDE>(device, stream, p, r, ctas);
    case 256: return backward_ring<DT, 256, 4, WIDE>(device, stream, p, r, ctas);
    case 384: return backward_ring<DT, 384, 4, WIDE>(device, stream, p, r, ctas);
    default: return backward_ring<DT, 512, 4, WIDE>(device, stream, p, r, ctas);
  }
}

template <int DT, int T>
int forward_ring(int device, cudaStream_t stream, const NormParams& p) {
  auto kernel = layer_norm_ring_kernel<DT, T>;
  static bool configured[64] = {};
  if (!configured[device & 63]) {
    TVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingRoom));
    configured[device & 63] = true;
  }
  const int stages = std::min(kRingStages, kRingRoom / (p.d * 2));
  int* status = nullptr;
  if (status_word(device, &status) != 0) return -1;
  const int64_t ctas = std::min<int64_t>(sm_count(device), p.rows);
  return launch_dependent("layer_norm_ring", kernel, dim3(static_cast<unsigned>(ctas)), dim3(T), static_cast<size_t>(stages) * p.d * 2, stream, p,
                          stages, status);
}

template <int DT>
int forward(int device, cudaStream_t stream, const NormParams& p) {
  constexpr int kVec = DT == TVB_F32 ? 4 : 8;
  if (p.d > kLongest)
    return launch_dependent("layer_norm_long", layer_norm_long_kernel<DT>, dim3(static_cast<unsigned>(p.rows)), dim3(1024), 0, stream, p);
  // 16-byte accesses where every row of every operand begins on 16 bytes
  const bool vec = p.d % kVec == 0 && p.x_ld % kVec == 0 && aligned16(p.x) && aligned16(p.y) && aligned16(p.weight) && aligned16(p.bias);
  if constexpr (DT != TVB_F32) {
    const bool wide = p.param_dtype == TVB_F32 && (p.weight != nullptr || p.bias != nullptr);
    if (vec && !wide && p.d > 8 * 1024 && p.d <= 16 * 1024)
      return p.d <= 32 * 384 ? forward_ring<DT, 384>(device, stream, p) : forward_ring<DT, 512>(device, stream, p);
  }
  return vec ? forward_vec<DT, kVec>(stream, p) : forward_vec<DT, 1>(stream, p);
}

// Queues the kernels of dx and of the partial sums; *parts receives the number of partial rows.
template <int DT>
int backward(int device, cudaStream_t stream, const NormParams& p, int64_t* parts) {
  constexpr int kVec = DT == TVB_F32 ? 4 : 8;
  const bool vec = p.d % kVec == 0 && p.x_ld % kVec == 0 && p.dy_ld % kVec == 0 && aligned16(p.x) && aligned16(p.dy) &&
                   aligned16(p.y) && aligned16(p.weight) && aligned16(p.partial);
  const bool wide = DT == TVB_F32 || (p.param_dtype == TVB_F32 && p.weight != nullptr);
  const Ring ring = vec ? ring_shape(p.d, DT == TVB_F32 ? 4 : 2, wide) : Ring{};
  if (ring.stages != 0) {
    const int64_t ctas = ring_ctas(p.rows, ring);
    *parts = ctas / kRingCluster;
    if constexpr (DT != TVB_F32) {
      if (!wide) return backward_ring_threads<DT, false>(device, stream, p, ring, ctas);
    }
    return backward_ring_threads<DT, true>(device, stream, p, ring, ctas);
  }
  *parts = norm_parts(p.rows, p.d);
  if (p.d > kLongestBwd) {
    if (p.y != nullptr && launch_dependent("layer_norm_backward_long", layer_norm_backward_long_kernel<DT>,
                                           dim3(static_cast<unsigned>(p.rows)), dim3(1024), 0, stream, p) != 0)
      return -1;
    if (p.partial == nullptr) return 0;
    return launch_dependent("layer_norm_columns", layer_norm_columns_kernel<DT>,
                            dim3(static_cast<unsigned>(ceil_div(p.d, 256)), static_cast<unsigned>(*parts)), dim3(256), 0, stream, p);
  }
  return vec ? backward_vec<DT, kVec>(stream, p, *parts) : backward_vec<DT, 1>(stream, p, *parts);
}

int check_sizes(const char* fn, int dtype, int param_dtype, int64_t rows, int64_t d) {
  auto is_float = [](int dt) { return dt == TVB_F32 || dt == TVB_F16 || dt == TVB_BF16; };
  TVB_REQUIRE(is_float(dtype), std::string(fn) + ": x must be float32, float16 or bfloat16");
  TVB_REQUIRE(param_dtype == dtype || param_dtype == TVB_F32, std::string(fn) + ": weight and bias must be of x's dtype or float32");
  TVB_REQUIRE(rows >= 0 && d >= 0, std::string(fn) + ": negative size");
  TVB_REQUIRE(rows < (int64_t(1) << 31) && d < (int64_t(1) << 30), std::string(fn) + ": more than 2^31 - 1 rows or 2^30 - 1 values per row");
  return 0;
}

}  // namespace
}  // namespace tvb

using namespace tvb;

extern "C" int tvb_layer_norm(int device, const void* x, int dtype, int64_t x_sm, const void* weight, const void* bias, int param_dtype,
                              float eps, void* y, float* mean, float* rstd, int64_t rows, int64_t d, void* caller_stream) {
  if (check_sizes("tvb_layer_norm", dtype, param_dtype, rows, d) != 0) return -1;
  TVB_REQUIRE(eps >= 0.0f, "tvb_layer_norm: eps must not be negative");
  TVB_REQUIRE(rows <= 1 || x_sm >= d, "tvb_layer_norm: rows of x must be at least d apart");
  if (rows == 0 || d == 0) return 0;
  TVB_REQUIRE(x != nullptr && y != nullptr, "tvb_layer_norm: NULL pointer");
  const int64_t es = dtype_size(dtype), x_bytes = ((rows - 1) * x_sm + d) * es, p_bytes = d * dtype_size(param_dtype);
  const void* outs[3] = {y, mean, rstd};
  const int64_t out_bytes[3] = {rows * d * es, rows * 4, rows * 4};
  for (int i = 0; i < 3; i++) {
    TVB_REQUIRE(!overlap(outs[i], out_bytes[i], x, x_bytes) && !overlap(outs[i], out_bytes[i], weight, p_bytes) &&
                    !overlap(outs[i], out_bytes[i], bias, p_bytes),
                "tvb_layer_norm: an output overlaps an operand");
    for (int j = 0; j < i; j++)
      TVB_REQUIRE(!overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]), "tvb_layer_norm: one output overlaps another");
  }
  cudaStream_t stream;
  if (enter_on(device, caller_stream, &stream) != 0) return -1;
  NormParams p{};
  p.x = x; p.weight = weight; p.bias = bias; p.y = y; p.mean = mean; p.rstd = rstd;
  p.x_ld = rows > 1 ? x_sm : d;
  p.rows = rows; p.d = static_cast<int>(d); p.param_dtype = param_dtype; p.eps = eps;
  if (dtype == TVB_F32) return forward<TVB_F32>(device, stream, p);
  if (dtype == TVB_F16) return forward<TVB_F16>(device, stream, p);
  return forward<TVB_BF16>(device, stream, p);
}

extern "C" uint64_t tvb_layer_norm_backward_workspace_bytes(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0) return 0;
  const Ring ring = ring_shape(d, 2, false);  // (wider rows take as many CTAs or none)
  const int64_t most = std::max(norm_parts(rows, d), ring.stages != 0 ? ring_ctas(rows, ring) / kRingCluster : 0);
  return static_cast<uint64_t>(most) * 2 * static_cast<uint64_t>(d) * 4;
}

extern "C" int tvb_layer_norm_backward(int device, const void* dy, int dtype, int64_t dy_sm, const void* x, int64_t x_sm,
                                       const float* mean, const float* rstd, const void* weight, int param_dtype, void* dx, void* dweight,
                                       void* dbias, int64_t rows, int64_t d, void* workspace, uint64_t workspace_bytes,
                                       void* caller_stream) {
  if (check_sizes("tvb_layer_norm_backward", dtype, param_dtype, rows, d) != 0) return -1;
  TVB_REQUIRE(rows <= 1 || (x_sm >= d && dy_sm >= d), "tvb_layer_norm_backward: rows of x and dy must be at least d apart");
  if (d == 0 || (dx == nullptr && dweight == nullptr && dbias == nullptr)) return 0;
  const bool sums = dweight != nullptr || dbias != nullptr;
  TVB_REQUIRE(rows == 0 || (dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr), "tvb_layer_norm_backward: NULL pointer");
  const uint64_t need = sums ? tvb_layer_norm_backward_workspace_bytes(rows, d) : 0;
  TVB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && aligned16(workspace)),
              "tvb_layer_norm_backward: the workspace is too small or not 16-byte aligned");
  const int64_t es = dtype_size(dtype), ps = dtype_size(param_dtype) * d;
  const int64_t x_bytes = rows == 0 ? 0 : ((rows - 1) * x_sm + d) * es, dy_bytes = rows == 0 ? 0 : ((rows - 1) * dy_sm + d) * es;
  const void* outs[4] = {dx, dweight, dbias, need != 0 ? workspace : nullptr};
  const int64_t out_bytes[4] = {rows * d * es, ps, ps, static_cast<int64_t>(need)};
  for (int i = 0; i < 4; i++) {
    TVB_REQUIRE(!overlap(outs[i], out_bytes[i], x, x_bytes) && !overlap(outs[i], out_bytes[i], dy, dy_bytes) &&
                    !overlap(outs[i], out_bytes[i], mean, rows * 4) && !overlap(outs[i], out_bytes[i], rstd, rows * 4) &&
                    !overlap(outs[i], out_bytes[i], weight, ps),
                "tvb_layer_norm_backward: an output or the workspace overlaps an operand");
    for (int j = 0; j < i; j++)
      TVB_REQUIRE(!overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]), "tvb_layer_norm_backward: two outputs overlap");
  }
  cudaStream_t stream;
  if (enter_on(device, caller_stream, &stream) != 0) return -1;
  NormParams p{};
  p.x = x; p.dy = dy; p.weight = weight; p.y = dx;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
  p.x_ld = rows > 1 ? x_sm : d;
  p.dy_ld = rows > 1 ? dy_sm : d;
  p.rows = rows; p.d = static_cast<int>(d); p.param_dtype = param_dtype;
  int64_t parts = 0;
  if (rows > 0) {
    const int rc = dtype == TVB_F32   ? backward<TVB_F32>(device, stream, p, &parts)
                   : dtype == TVB_F16 ? backward<TVB_F16>(device, stream, p, &parts)
                                      : backward<TVB_BF16>(device, stream, p, &parts);
    if (rc != 0) return -1;
  }
  if (!sums) return 0;
  return launch_dependent("layer_norm_reduce", layer_norm_reduce_kernel, dim3(static_cast<unsigned>(ceil_div(2 * d, 32))), dim3(256), 0,
                          stream, p.partial, static_cast<int>(parts), p.d, dweight, dbias, param_dtype);
}
