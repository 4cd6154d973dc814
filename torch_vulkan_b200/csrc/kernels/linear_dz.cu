// dz = dy * act'(z) and db = the sums of dz over the rows, in one pass over dy and z.
//
// A cluster of CTAs owns a strip of 64 columns; each of its CTAs takes a contiguous share of the rows, 32 at a time, eight
// neighbouring threads covering a row's strip. The sums stay in float32 (of the unrounded dz): per thread in registers, per
// CTA through shared memory, per cluster through distributed shared memory, always in the same order, so db repeats bit for
// bit and needs neither atomics nor a workspace.
#include <cooperative_groups.h>

#include "../core/common.h"
#include "launch.h"
#include "linear.h"
#include "linear_epilogue.cuh"
#include "numerics.cuh"
#include "ptx.cuh"

namespace tvb {
namespace {

constexpr int kStrip = 64, kThreads = 256, kRowsPerStep = 32;

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, float (&v)[8]) {
  if constexpr (DT == TVB_F32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    const float4 a = s[0], b = s[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 t = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float2 f = unpack16<DT == TVB_BF16>(w[e]);
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t i, const float (&v)[8]) {
  if constexpr (DT == TVB_F32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    constexpr bool kB = DT == TVB_BF16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) =
        make_uint4(pack16<kB>(v[0], v[1]), pack16<kB>(v[2], v[3]), pack16<kB>(v[4], v[5]), pack16<kB>(v[6], v[7]));
  }
}

// v *= act'(z), the choice of activation made once for the eight.
template <bool FAST>
__device__ __forceinline__ void slopes8(float (&v)[8], const float (&z)[8], int act) {
  switch (act) {
    case TVB_ACT_RELU:
#pragma unroll
      for (int c = 0; c < 8; c++) v[c] *= act_slope<FAST>(z[c], TVB_ACT_RELU);
      break;
    case TVB_ACT_GELU:
#pragma unroll
      for (int c = 0; c < 8; c++) v[c] *= act_slope<FAST>(z[c], TVB_ACT_GELU);
      break;
    case TVB_ACT_GELU_TANH:
#pragma unroll
      for (int c = 0; c < 8; c++) v[c] *= act_slope<FAST>(z[c], TVB_ACT_GELU_TANH);
      break;
    default:
#pragma unroll
      for (int c = 0; c < 8; c++) v[c] *= act_slope<FAST>(z[c], TVB_ACT_SILU);
      break;
  }
}

// VEC: dy, z and dz are read and written 16 bytes at a time (8 values of 16 bits, 4 of 32, twice).
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) linear_dz_kernel(const LinearDz p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int64_t c0 = static_cast<int64_t>(blockIdx.x / parts) * kStrip + (threadIdx.x & 7) * 8;
  const int64_t r_begin = p.m * part / parts, r_end = p.m * (part + 1) / parts;
  const bool act = p.activation != TVB_ACT_NONE;
  float sum[8] = {};
  if (VEC) {
    if (c0 < p.n) {
#pragma unroll 2
      for (int64_t r = r_begin + (threadIdx.x >> 3); r < r_end; r += kRowsPerStep) {
        float v[8], z[8];
        load8<DT>(p.dy, r * p.dy_ld + c0, v);
        if (act) {
          load8<DT>(p.z, r * p.n + c0, z);
          slopes8<DT != TVB_F32>(v, z, p.activation);
        }
#pragma unroll
        for (int c = 0; c < 8; c++) sum[c] += v[c];
        if (p.dz != nullptr) store8<DT>(p.dz, r * p.dz_ld + c0, v);
      }
    }
  } else {
    for (int64_t r = r_begin + (threadIdx.x >> 3); r < r_end; r += kRowsPerStep) {
#pragma unroll
      for (int c = 0; c < 8; c++) {
        if (c0 + c >= p.n) break;
        float v = load_float<DT>(p.dy, r * p.dy_ld + c0 + c);
        if (act) v *= act_slope<DT != TVB_F32>(load_float<DT>(p.z, r * p.n + c0 + c), p.activation);
        sum[c] += v;
        if (p.dz != nullptr) store_float<DT>(p.dz, r * p.dz_ld + c0 + c, v);
      }
    }
  }
  __shared__ float part_sums[kRowsPerStep][kStrip];
  __shared__ float cta_sums[kStrip];
#pragma unroll
  for (int c = 0; c < 8; c++) part_sums[threadIdx.x >> 3][(threadIdx.x & 7) * 8 + c] = sum[c];
  __syncthreads();
  if (threadIdx.x < kStrip) {
    float s = 0.0f;
    for (int g = 0; g < kRowsPerStep; g++) s += part_sums[g][threadIdx.x];
    cta_sums[threadIdx.x] = s;
  }
  cluster.sync();
  const int64_t col = static_cast<int64_t>(blockIdx.x / parts) * kStrip + threadIdx.x;
  if (part == 0 && threadIdx.x < kStrip && col < p.n && p.db != nullptr) {
    float s = 0.0f;
    for (int g = 0; g < parts; g++) s += *cluster.map_shared_rank(&cta_sums[threadIdx.x], g);
    store_float<DT>(p.db, col, s);
  }
  cluster.sync();
}

// Rows that begin anywhere brought to rows that begin on 16 bytes: eight values per thread, one or two matrices per launch.
__global__ void __launch_bounds__(kThreads) linear_copy_kernel(const LinearCopy a, const LinearCopy b) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int64_t per_a = a.dst_ld / 8, total_a = a.rows * per_a, per_b = b.dst_ld / 8, total = total_a + b.rows * per_b;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; e < total; e += static_cast<int64_t>(gridDim.x) * kThreads) {
    const bool first = e < total_a;
    const LinearCopy& d = first ? a : b;
    const int64_t x = first ? e : e - total_a, per = first ? per_a : per_b;
    const int64_t r = x / per, c = (x - r * per) * 8;
    const uint16_t* src = static_cast<const uint16_t*>(d.src) + r * d.src_ld + c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t lo = c + 2 * j < d.cols ? src[2 * j] : 0u, hi = c + 2 * j + 1 < d.cols ? src[2 * j + 1] : 0u;
      w[j] = lo | (hi << 16);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(d.dst) + r * d.dst_ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace

int linear_copy(int device, cudaStream_t stream, const LinearCopy& a, const LinearCopy& b) {
  const int64_t want = ceil_div(a.rows * (a.dst_ld / 8) + b.rows * (b.dst_ld / 8), kThreads), most = static_cast<int64_t>(sm_count(device)) * 16;
  if (want == 0) return 0;
  return launch_dependent("linear_copy", linear_copy_kernel, dim3(static_cast<unsigned>(std::min(want, most))), dim3(kThreads), 0, stream, a, b);
}

int linear_dz(int device, cudaStream_t stream, const LinearDz& p) {
  const int64_t strips = ceil_div(p.n, kStrip);
  // as many CTAs per strip as have four steps of rows to do, until the GPU is full
  int parts = 1;
  while (parts < 8 && p.m >= static_cast<int64_t>(parts) * 2 * kRowsPerStep * 4 && strips * parts < 4ll * sm_count(device)) parts *= 2;
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool vec = p.n % 8 == 0 && p.dy_ld % 8 == 0 && p.dz_ld % 8 == 0 && aligned(p.dy) && aligned(p.dz) && (p.activation == TVB_ACT_NONE || aligned(p.z));
  auto kernel = p.dtype == TVB_F32   ? (vec ? linear_dz_kernel<TVB_F32, true> : linear_dz_kernel<TVB_F32, false>)
                : p.dtype == TVB_F16 ? (vec ? linear_dz_kernel<TVB_F16, true> : linear_dz_kernel<TVB_F16, false>)
                                     : (vec ? linear_dz_kernel<TVB_BF16, true> : linear_dz_kernel<TVB_BF16, false>);
  return launch_dependent_cluster("linear_dz", kernel, parts, dim3(static_cast<unsigned>(strips * parts)), dim3(kThreads), 0, stream, p);
}

}  // namespace tvb
