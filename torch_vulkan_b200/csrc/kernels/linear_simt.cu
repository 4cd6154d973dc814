// The products of linear.h in float32, on the CUDA cores, for any strides: 64 x 64 tiles, float32 sums.
#include "../core/common.h"
#include "linear.h"
#include "linear_math.cuh"
#include "numerics.cuh"

namespace tvb {
namespace {

constexpr int kTile = 64, kStep = 16;

__global__ void __launch_bounds__(256) linear_simt_kernel(const LinearProduct p) {
  __shared__ float ps[kStep][kTile + 1], qs[kStep][kTile + 1];
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTile, j0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t r0 = 0; r0 < p.R; r0 += kStep) {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      // neighbouring threads read along whichever stride is 1
      const int e = threadIdx.x + 256 * u;
      const int pi = !p.p_mn ? e >> 4 : e & 63, pr = !p.p_mn ? e & 15 : e >> 6;
      const int qj = !p.q_mn ? e >> 4 : e & 63, qr = !p.q_mn ? e & 15 : e >> 6;
      ps[pr][pi] = i0 + pi < p.I && r0 + pr < p.R ? load_float<TVB_F32>(p.p, (i0 + pi) * p.p_si + (r0 + pr) * p.p_sr) : 0.0f;
      qs[qr][qj] = j0 + qj < p.J && r0 + qr < p.R ? load_float<TVB_F32>(p.q, (j0 + qj) * p.q_sj + (r0 + qr) * p.q_sr) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kStep; r++) {
      float pv[4], qv[4];
#pragma unroll
      for (int a = 0; a < 4; a++) {
        pv[a] = ps[r][tx + 16 * a];
        qv[a] = qs[r][ty + 16 * a];
      }
#pragma unroll
      for (int a = 0; a < 4; a++)
#pragma unroll
        for (int b = 0; b < 4; b++) acc[a][b] = fmaf(pv[b], qv[a], acc[a][b]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int a = 0; a < 4; a++) {
    const int64_t j = j0 + ty + 16 * a;
    if (j >= p.J) continue;
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int64_t i = i0 + tx + 16 * b;
      if (i >= p.I) continue;
      float z = acc[a][b];
      if (p.bias != nullptr) z += load_float<TVB_F32>(p.bias, i);
      if (p.preact != nullptr) store_float<TVB_F32>(p.preact, j * p.I + i, z);
      float y = act_value(z, p.activation);
      if (p.residual != nullptr) y += load_float<TVB_F32>(p.residual, j * p.residual_ld + i);
      store_float<TVB_F32>(p.out, j * p.I + i, y);
    }
  }
}

}  // namespace

int linear_simt(cudaStream_t stream, const LinearProduct& p) {
  const int64_t rows = ceil_div(p.J, kTile);
  if (rows > 65535) return fail("tvb_linear: too many rows for one launch of the CUDA-core kernel (4194240)");
  const dim3 grid(static_cast<unsigned>(ceil_div(p.I, kTile)), static_cast<unsigned>(rows));
  linear_simt_kernel<<<grid, 256, 0, stream>>>(p);
  return launched("linear_simt", grid, dim3(256), 0, stream);
}

}  // namespace tvb
