// Layer norm over the last dimension, forward and backward:
//   y = (x - mean) rstd g + b,   mean = <x>,   rstd = 1 / sqrt(<(x - mean)^2> + eps)        <.> the mean over a row
//   dx = rstd (u - <u> - h <u h>),   u = dy g,  h = (x - mean) rstd
//   dg = sum over rows of dy h,   db = sum over rows of dy
//
// Bound by memory: the forward pass reads and writes a row once, the backward pass reads two rows and writes one. A group of T
// threads (8 or 32 of a warp, or a whole CTA) keeps its row in registers between the statistics and the result, so a row
// is read once; the variance is taken from the centred values (two passes over registers, none over memory), which a
// mean far from zero does not spoil. All statistics and sums are float32.
// The backward pass keeps the sums of dg and db of its columns in registers over all rows that the group handles; one
// partial row per CTA goes to the workspace and a second kernel adds those in a fixed order (no atomics: the gradients
// repeat bit for bit).
#include "../core/common.h"
#include "launch.h"
#include "linear_math.cuh"
#include "numerics.cuh"
#include "ptx.cuh"

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

// Sums over the T threads of a group; every thread gets them. `slot` alternates between calls (two buffers: one barrier
// per call is then enough).
template <int T>
__device__ __forceinline__ void group_sum(float& a, float& b, float2 (*buf)[32], int slot) {
#pragma unroll
  for (int s = (T < 32 ? T : 32) / 2; s > 0; s >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, s);
    b += __shfl_xor_sync(0xffffffffu, b, s);
  }
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) buf[slot][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = 0.0f;
    b = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 32; w++) {
      const float2 v = buf[slot][w];
      a += v.x;
      b += v.y;
    }
  }
}

template <int T>
constexpr int norm_threads() { return T < 128 ? 128 : T; }

constexpr int kVals = 32;      // values of a row per thread, forward
constexpr int kValsBwd = 16;   // backward (with two sums per value beside them)

template <int DT, int VEC, int T>
__global__ void __launch_bounds__(norm_threads<T>()) layer_norm_kernel(const NormParams p) {
  constexpr int kChunks = kVals / VEC, kGroups = norm_threads<T>() / T;
  __shared__ float2 buf[2][32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int t = threadIdx.x % T;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / T;
  const bool live = row < p.rows;  // (every thread takes part in the shuffles)
  float x[kChunks][VEC];
  float sum = 0.0f, none = 0.0f;
#pragma unroll
  for (int c = 0; c < kChunks; c++) {
    const int col = (c * T + t) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; j++) x[c][j] = 0.0f;
    if (live && col < p.d) load_vec<DT, VEC>(p.x, row * p.x_ld + col, x[c]);
  }
#pragma unroll
  for (int c = 0; c < kChunks; c++)
#pragma unroll
    for (int j = 0; j < VEC; j++) sum += x[c][j];
  group_sum<T>(sum, none, buf, 0);
  const float mean = sum / static_cast<float>(p.d);
  float sq = 0.0f;
#pragma unroll
  for (int c = 0; c < kChunks; c++)
    if ((c * T + t) * VEC < p.d) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        x[c][j] -= mean;
        sq = fmaf(x[c][j], x[c][j], sq);
      }
    }
  group_sum<T>(sq, none, buf, 1);
  const float rstd = 1.0f / sqrtf(sq / static_cast<float>(p.d) + p.eps);
  if (!live) return;
  if (t == 0) {
    if (p.mean != nullptr) p.mean[row] = mean;
    if (p.rstd != nullptr) p.rstd[row] = rstd;
  }
#pragma unroll
  for (int c = 0; c < kChunks; c++) {
    const int col = (c * T + t) * VEC;
    if (col >= p.d) continue;
    float g[VEC], b[VEC];
    load_param<DT, VEC>(p.weight, p.param_dtype, col, 1.0f, g);
    load_param<DT, VEC>(p.bias, p.param_dtype, col, 0.0f, b);
#pragma unroll
    for (int j = 0; j < VEC; j++) g[j] = fmaf(x[c][j] * rstd, g[j], b[j]);
    store_vec<DT, VEC>(p.y, row * p.d + col, g);
  }
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

constexpr int kLongest = 32 * 1024;         // values of a row that the forward kernel keeps in registers
constexpr int kLongestBwd = 16 * 1024;
constexpr int64_t kLongSlices = 64;         // partial rows of layer_norm_columns_kernel, at most

int norm_group(int64_t d, int vals) {
  for (int t : {8, 32, 128, 256, 512})
    if (d <= static_cast<int64_t>(t) * vals) return t;
  return 1024;
}

// CTAs of the backward kernel (and partial rows of its sums).
int64_t norm_parts(int64_t rows, int64_t d) {
  if (d > kLongestBwd) return std::min<int64_t>(rows, kLongSlices);
  const int t = norm_group(d, kValsBwd);
  const int64_t groups = t < 128 ? 128 / t : 1;
  const int64_t most = t <= 128 ? 148 * 4 : (t == 256 ? 148 * 2 : 148);
  return std::min(ceil_div(rows, groups), most);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int DT, int VEC>
int forward_vec(cudaStream_t stream, const NormParams& p) {
  const int t = norm_group(p.d, kVals);
  const int64_t grid = t < 128 ? ceil_div(p.rows, 128 / t) : p.rows;
  auto kernel = t == 8 ? layer_norm_kernel<DT, VEC, 8> : t == 32 ? layer_norm_kernel<DT, VEC, 32> : t == 128 ? layer_norm_kernel<DT, VEC, 128>
              : t == 256 ? layer_norm_kernel<DT, VEC, 256> : t == 512 ? layer_norm_kernel<DT, VEC, 512> : layer_norm_kernel<DT, VEC, 1024>;
  return launch_dependent("layer_norm", kernel, dim3(static_cast<unsigned>(grid)), dim3(t < 128 ? 128 : t), 0, stream, p);
}

template <int DT, int VEC>
int backward_vec(cudaStream_t stream, const NormParams& p, int64_t parts) {
  const int t = norm_group(p.d, kValsBwd);
  auto kernel = t == 8 ? layer_norm_backward_kernel<DT, VEC, 8> : t == 32 ? layer_norm_backward_kernel<DT, VEC, 32>
              : t == 128 ? layer_norm_backward_kernel<DT, VEC, 128> : t == 256 ? layer_norm_backward_kernel<DT, VEC, 256>
              : t == 512 ? layer_norm_backward_kernel<DT, VEC, 512> : layer_norm_backward_kernel<DT, VEC, 1024>;
  return launch_dependent("layer_norm_backward", kernel, dim3(static_cast<unsigned>(parts)), dim3(t < 128 ? 128 : t), 0, stream, p);
}

template <int DT>
int forward(cudaStream_t stream, const NormParams& p) {
  constexpr int kVec = DT == TVB_F32 ? 4 : 8;
  if (p.d > kLongest)
    return launch_dependent("layer_norm_long", layer_norm_long_kernel<DT>, dim3(static_cast<unsigned>(p.rows)), dim3(1024), 0, stream, p);
  // 16-byte accesses where every row of every operand begins on 16 bytes
  const bool vec = p.d % kVec == 0 && p.x_ld % kVec == 0 && aligned16(p.x) && aligned16(p.y) && aligned16(p.weight) && aligned16(p.bias);
  return vec ? forward_vec<DT, kVec>(stream, p) : forward_vec<DT, 1>(stream, p);
}

template <int DT>
int backward(cudaStream_t stream, const NormParams& p, int64_t parts) {
  constexpr int kVec = DT == TVB_F32 ? 4 : 8;
  if (p.d > kLongestBwd) {
    if (p.y != nullptr && launch_dependent("layer_norm_backward_long", layer_norm_backward_long_kernel<DT>,
                                           dim3(static_cast<unsigned>(p.rows)), dim3(1024), 0, stream, p) != 0)
      return -1;
    if (p.partial == nullptr) return 0;
    return launch_dependent("layer_norm_columns", layer_norm_columns_kernel<DT>,
                            dim3(static_cast<unsigned>(ceil_div(p.d, 256)), static_cast<unsigned>(parts)), dim3(256), 0, stream, p);
  }
  const bool vec = p.d % kVec == 0 && p.x_ld % kVec == 0 && p.dy_ld % kVec == 0 && aligned16(p.x) && aligned16(p.dy) &&
                   aligned16(p.y) && aligned16(p.weight);
  return vec ? backward_vec<DT, kVec>(stream, p, parts) : backward_vec<DT, 1>(stream, p, parts);
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
  const int64_t es = dtype_size(dtype), x_bytes = ((rows - 1) * x_sm + d) * es, y_bytes = rows * d * es;
  TVB_REQUIRE(!overlap(y, y_bytes, x, x_bytes) && !overlap(mean, rows * 4, x, x_bytes) && !overlap(rstd, rows * 4, x, x_bytes) &&
                  !overlap(mean, rows * 4, y, y_bytes) && !overlap(rstd, rows * 4, y, y_bytes) && !overlap(mean, rows * 4, rstd, rows * 4) &&
                  !overlap(y, y_bytes, weight, d * dtype_size(param_dtype)) && !overlap(y, y_bytes, bias, d * dtype_size(param_dtype)),
              "tvb_layer_norm: an output overlaps another operand");
  cudaStream_t stream;
  if (enter_on(device, caller_stream, &stream) != 0) return -1;
  NormParams p{};
  p.x = x; p.weight = weight; p.bias = bias; p.y = y; p.mean = mean; p.rstd = rstd;
  p.x_ld = rows > 1 ? x_sm : d;
  p.rows = rows; p.d = static_cast<int>(d); p.param_dtype = param_dtype; p.eps = eps;
  if (dtype == TVB_F32) return forward<TVB_F32>(stream, p);
  if (dtype == TVB_F16) return forward<TVB_F16>(stream, p);
  return forward<TVB_BF16>(stream, p);
}

extern "C" uint64_t tvb_layer_norm_backward_workspace_bytes(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0) return 0;
  return static_cast<uint64_t>(norm_parts(rows, d)) * 2 * static_cast<uint64_t>(d) * 4;
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
  const int64_t parts = rows > 0 ? norm_parts(rows, d) : 0;
  if (rows > 0) {
    const int rc = dtype == TVB_F32 ? backward<TVB_F32>(stream, p, parts) : dtype == TVB_F16 ? backward<TVB_F16>(stream, p, parts)
                                                                                               : backward<TVB_BF16>(stream, p, parts);
    if (rc != 0) return -1;
  }
  if (!sums) return 0;
  return launch_dependent("layer_norm_reduce", layer_norm_reduce_kernel, dim3(static_cast<unsigned>(ceil_div(2 * d, 32))), dim3(256), 0,
                          stream, p.partial, static_cast<int>(parts), p.d, dweight, dbias, param_dtype);
}
