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

// Eight neighbouring values as four pairs.
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, uint64_t (&v)[4]) {
  if constexpr (DT == TVB_F32) {
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
    const uint4 a = s[0], b = s[1];
    v[0] = ptx::pack_f32x2(a.x, a.y); v[1] = ptx::pack_f32x2(a.z, a.w); v[2] = ptx::pack_f32x2(b.x, b.y); v[3] = ptx::pack_f32x2(b.z, b.w);
  } else {
    constexpr bool kB = DT == TVB_BF16;
    const uint4 t = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    v[0] = unpack16<kB>(t.x); v[1] = unpack16<kB>(t.y); v[2] = unpack16<kB>(t.z); v[3] = unpack16<kB>(t.w);
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t i, const uint64_t (&v)[4]) {
  if constexpr (DT == TVB_F32) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; e++) ptx::unpack_f32x2(v[e], f[2 * e], f[2 * e + 1]);
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    d[0] = make_float4(f[0], f[1], f[2], f[3]);
    d[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    constexpr bool kB = DT == TVB_BF16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) = make_uint4(pack16<kB>(v[0]), pack16<kB>(v[1]), pack16<kB>(v[2]), pack16<kB>(v[3]));
  }
}

// v *= act'(z)
template <int DT>
__device__ __forceinline__ void times_slope(uint64_t (&v)[4], const uint64_t (&z)[4], int act) {
  if constexpr (DT == TVB_F32) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float a, b;
      ptx::unpack_f32x2(z[e], a, b);
      v[e] = ptx::mul_f32x2(v[e], ptx::pack_f32x2(__float_as_uint(act_slope(a, act)), __float_as_uint(act_slope(b, act))));
    }
  } else {
    times_slope_pairs(v, z, act);
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
  uint64_t sum[4] = {};
  const int64_t c_end = p.n - c0;  // columns of this thread that exist
  // kAhead rows are read before the first is worked on: a store between two loads would hold the second back
  constexpr int kAhead = VEC && DT != TVB_F32 ? 4 : 2;
  auto one = [&](int64_t r, uint64_t (&v)[4], const uint64_t (&z)[4]) {
    if (act) times_slope<DT>(v, z, p.activation);
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] = ptx::add_f32x2(sum[e], v[e]);
    if (p.dz == nullptr) return;
    if (VEC) {
      store8<DT>(p.dz, r * p.dz_ld + c0, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float f[2];
        ptx::unpack_f32x2(v[e], f[0], f[1]);
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (2 * e + h < c_end) store_float<DT>(p.dz, r * p.dz_ld + c0 + 2 * e + h, f[h]);
      }
    }
  };
  auto fetch = [&](int64_t r, uint64_t (&v)[4], uint64_t (&z)[4]) {
    if (VEC) {
      load8<DT>(p.dy, r * p.dy_ld + c0, v);
      if (act) load8<DT>(p.z, r * p.n + c0, z);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float f[4] = {};
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (2 * e + h < c_end) {
            f[h] = load_float<DT>(p.dy, r * p.dy_ld + c0 + 2 * e + h);
            if (act) f[2 + h] = load_float<DT>(p.z, r * p.n + c0 + 2 * e + h);
          }
        v[e] = ptx::pack_f32x2(__float_as_uint(f[0]), __float_as_uint(f[1]));
        z[e] = ptx::pack_f32x2(__float_as_uint(f[2]), __float_as_uint(f[3]));
      }
    }
  };
  if (c_end > 0) {
    int64_t r = r_begin + (threadIdx.x >> 3);
    uint64_t v[kAhead][4], z[kAhead][4] = {};
    for (; r + (kAhead - 1) * kRowsPerStep < r_end; r += kAhead * kRowsPerStep) {
#pragma unroll
      for (int a = 0; a < kAhead; a++) fetch(r + a * kRowsPerStep, v[a], z[a]);
#pragma unroll
      for (int a = 0; a < kAhead; a++) one(r + a * kRowsPerStep, v[a], z[a]);
    }
    for (; r < r_end; r += kRowsPerStep) {
      fetch(r, v[0], z[0]);
      one(r, v[0], z[0]);
    }
  }
  __shared__ float part_sums[kRowsPerStep][kStrip];
  __shared__ float cta_sums[kStrip];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    float lo, hi;
    ptx::unpack_f32x2(sum[e], lo, hi);
    part_sums[threadIdx.x >> 3][(threadIdx.x & 7) * 8 + 2 * e] = lo;
    part_sums[threadIdx.x >> 3][(threadIdx.x & 7) * 8 + 2 * e + 1] = hi;
  }
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
