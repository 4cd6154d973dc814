// dz = dy * act'(z) and db = the sums of dz over the rows, in one pass over dy and z.
//
// A cluster of CTAs owns a strip of 64 columns; each of its CTAs takes a contiguous share of the rows, 32 at a time, eight
// neighbouring threads covering a row's strip. The sums stay in float32 (of the unrounded dz): per thread in registers, per
// CTA through shared memory, per cluster through distributed shared memory, always in the same order, so db repeats bit for
// bit and needs neither atomics nor a workspace.
#include <cooperative_groups.h>

#include "../core/common.h"
#include "linear.h"
#include "linear_math.cuh"
#include "numerics.cuh"

namespace tvb {
namespace {

constexpr int kStrip = 64, kThreads = 256, kRowsPerStep = 32;

template <int DT>
__global__ void __launch_bounds__(kThreads) linear_dz_kernel(const LinearDz p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int64_t c0 = static_cast<int64_t>(blockIdx.x / parts) * kStrip + (threadIdx.x & 7) * 8;
  const int64_t r_begin = p.m * part / parts, r_end = p.m * (part + 1) / parts;
  float sum[8] = {};
  for (int64_t r = r_begin + (threadIdx.x >> 3); r < r_end; r += kRowsPerStep) {
#pragma unroll
    for (int c = 0; c < 8; c++) {
      if (c0 + c >= p.n) break;
      float v = load_float<DT>(p.dy, r * p.dy_ld + c0 + c);
      if (p.activation != TVB_ACT_NONE) v *= act_slope<DT != TVB_F32>(load_float<DT>(p.z, r * p.n + c0 + c), p.activation);
      sum[c] += v;
      if (p.dz != nullptr) store_float<DT>(p.dz, r * p.dz_ld + c0 + c, v);
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

// Rows that begin anywhere brought to rows that begin on 16 bytes: eight values per thread.
__global__ void __launch_bounds__(kThreads) linear_pad_kernel(uint16_t* dst, int64_t dst_ld, const uint16_t* src, int64_t src_ld, int64_t rows,
                                                               int64_t cols) {
  const int64_t per_row = dst_ld / 8, total = rows * per_row;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; e < total; e += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = e / per_row, c = (e - r * per_row) * 8;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t lo = c + 2 * j < cols ? src[r * src_ld + c + 2 * j] : 0u, hi = c + 2 * j + 1 < cols ? src[r * src_ld + c + 2 * j + 1] : 0u;
      w[j] = lo | (hi << 16);
    }
    *reinterpret_cast<uint4*>(dst + r * dst_ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace

int linear_pad(int device, cudaStream_t stream, void* dst, int64_t dst_ld, const void* src, int64_t src_ld, int64_t rows, int64_t cols) {
  const int64_t want = ceil_div(rows * (dst_ld / 8), kThreads), most = static_cast<int64_t>(sm_count(device)) * 16;
  const int grid = static_cast<int>(std::min(want, most));
  linear_pad_kernel<<<grid, kThreads, 0, stream>>>(static_cast<uint16_t*>(dst), dst_ld, static_cast<const uint16_t*>(src), src_ld, rows, cols);
  return launched("linear_pad", dim3(grid), dim3(kThreads), 0, stream);
}

int linear_dz(int device, cudaStream_t stream, const LinearDz& p) {
  const int64_t strips = ceil_div(p.n, kStrip);
  // as many CTAs per strip as have four steps of rows to do, until the GPU is full
  int parts = 1;
  while (parts < 8 && p.m >= static_cast<int64_t>(parts) * 2 * kRowsPerStep * 4 && strips * parts < 4ll * sm_count(device)) parts *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(strips * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = p.dtype == TVB_F32 ? linear_dz_kernel<TVB_F32> : (p.dtype == TVB_F16 ? linear_dz_kernel<TVB_F16> : linear_dz_kernel<TVB_BF16>);
  TVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return launched("linear_dz", cfg.gridDim, cfg.blockDim, 0, stream);
}

}  // namespace tvb
