// The products of linear.h in float32, on the CUDA cores (the tensor cores have no float32).
//
// A CTA of eight warps makes a tile of 128 columns i and 8 WJ rows j: lane l holds columns 4 l .. 4 l + 3, a warp eight rows, and
// the 8 / WJ warps of the same rows take every (8 / WJ)-th r. Per r a lane reads a float4 of P and the warp's eight values of Q,
// which stand in shared memory twice each, as the operands of a two-float32 instruction: 16 of those against 5 loads. The next
// KSTEP values of r are on their way to registers meanwhile. With few tiles a cluster of CTAs cuts r into parts and joins its
// sums through distributed shared memory, in a fixed order.
//
// Few rows are bound by reading the weights (1 x 4096 x 14336: 87 us, 2.7 TB/s), many by the shared memory (2048 x 4096 x 4096:
// 2.1 ms, 33 TFLOP/s; tiles of 256 columns by two CTAs per SM spilled registers, 2.9 ms, by one 2.2).
#include "../core/common.h"
#include "launch.h"
#include "linear.h"
#include "linear_math.cuh"
#include "numerics.cuh"
#include "ptx_pair.cuh"

namespace tvb {
namespace {

constexpr int kThreads = 256, kWarps = 8;

template <int WJ, int KSTEP>
struct SimtCfg {
  static constexpr int kTI = 128, kTJ = 8 * WJ, kWR = kWarps / WJ;
  static constexpr int kPitchP = kTI, kPitchQ = 2 * kTJ + 4;
  // four rows r .. r + 3 of P have their float4s in an order of their own: neighbouring threads then write to different banks
  static constexpr int kTurn = KSTEP < 32 ? 32 / KSTEP : 1;
  static __device__ __forceinline__ int turn(int r4) { return (r4 * kTurn) & 7; }
  static constexpr int kRing = KSTEP * (kPitchP + kPitchQ) * 4, kSums = kWR * kTJ * kTI * 4;
  static constexpr int kSmem = kRing > kSums ? kRing : kSums;
  static constexpr int kLoadsP = KSTEP * kTI / 4 / kThreads, kLoadsQ = (KSTEP * kTJ / 4 + kThreads - 1) / kThreads;
};

// Four neighbouring values, `n` of which exist (the others are 0).
__device__ __forceinline__ float4 fetch4(const float* at, int64_t n, bool vec) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (vec && n >= 4) return *reinterpret_cast<const float4*>(at);
  if (n > 0) v.x = at[0];
  if (n > 1) v.y = at[1];
  if (n > 2) v.z = at[2];
  if (n > 3) v.w = at[3];
  return v;
}

__device__ __forceinline__ uint64_t both(float f) { return ptx::both_f32x2(f); }

template <int WJ, int KSTEP, bool P_MN, bool Q_MN>
__global__ void __launch_bounds__(kThreads, 2) linear_simt_kernel(const LinearProduct p, const uint32_t tiles_i, const int p_vec, const int q_vec) {
  using Cfg = SimtCfg<WJ, KSTEP>;
  constexpr int kTI = Cfg::kTI, kTJ = Cfg::kTJ, kWR = Cfg::kWR, kPitchP = Cfg::kPitchP, kPitchQ = Cfg::kPitchQ;
  extern __shared__ __align__(16) float smem[];
  float* ps = smem;
  float* qs = smem + KSTEP * kPitchP;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  uint32_t parts;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(parts));
  const uint32_t part = ptx::cluster_ctarank(), tile = blockIdx.x / parts;
  const int64_t i0 = static_cast<int64_t>(tile % tiles_i) * kTI, j0 = static_cast<int64_t>(tile / tiles_i) * kTJ;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, wj = warp % WJ, wr = warp / WJ;
  const int64_t steps = (p.R + KSTEP - 1) / KSTEP, s0 = steps * part / parts, s1 = steps * (part + 1) / parts;

  float4 np[Cfg::kLoadsP], nq[Cfg::kLoadsQ];
  auto fetch = [&](int64_t s) {
    const int64_t r0 = s * KSTEP;
#pragma unroll
    for (int u = 0; u < Cfg::kLoadsP; u++) {
      const int e = t + u * kThreads;
      const int64_t i = i0 + (P_MN ? e % (kTI / 4) * 4 : e / (KSTEP / 4)), r = r0 + (P_MN ? e / (kTI / 4) : e % (KSTEP / 4) * 4);
      const bool there = P_MN ? r < p.R : i < p.I;
      np[u] = fetch4(static_cast<const float*>(p.p) + (P_MN ? r * p.p_sr + i : i * p.p_si + r), there ? (P_MN ? p.I - i : p.R - r) : 0, p_vec);
    }
#pragma unroll
    for (int u = 0; u < Cfg::kLoadsQ; u++) {
      const int e = t + u * kThreads;
      const int64_t j = j0 + (Q_MN ? e % (kTJ / 4) * 4 : e / (KSTEP / 4)), r = r0 + (Q_MN ? e / (kTJ / 4) : e % (KSTEP / 4) * 4);
      const bool there = e < KSTEP * kTJ / 4 && (Q_MN ? r < p.R : j < p.J);
      nq[u] = fetch4(static_cast<const float*>(p.q) + (Q_MN ? r * p.q_sr + j : j * p.q_sj + r), there ? (Q_MN ? p.J - j : p.R - r) : 0, q_vec);
    }
  };
  auto stage = [&]() {
#pragma unroll
    for (int u = 0; u < Cfg::kLoadsP; u++) {
      const int e = t + u * kThreads;
      if (P_MN) {
        const int r = e / (kTI / 4);
        *reinterpret_cast<float4*>(ps + r * kPitchP + (e % (kTI / 4) ^ Cfg::turn(r >> 2)) * 4) = np[u];
      } else {
        const int r4 = e % (KSTEP / 4);
        float* d = ps + r4 * 4 * kPitchP + (e / (KSTEP / 4) ^ Cfg::turn(r4) * 4);
        d[0] = np[u].x; d[kPitchP] = np[u].y; d[2 * kPitchP] = np[u].z; d[3 * kPitchP] = np[u].w;
      }
    }
#pragma unroll
    for (int u = 0; u < Cfg::kLoadsQ; u++) {
      const int e = t + u * kThreads;
      if (e >= KSTEP * kTJ / 4) continue;
      if (Q_MN) {
        float4* d = reinterpret_cast<float4*>(qs + e / (kTJ / 4) * kPitchQ + e % (kTJ / 4) * 8);
        d[0] = make_float4(nq[u].x, nq[u].x, nq[u].y, nq[u].y);
        d[1] = make_float4(nq[u].z, nq[u].z, nq[u].w, nq[u].w);
      } else {
        float* d = qs + e % (KSTEP / 4) * 4 * kPitchQ + e / (KSTEP / 4) * 2;
        *reinterpret_cast<uint64_t*>(d) = both(nq[u].x);
        *reinterpret_cast<uint64_t*>(d + kPitchQ) = both(nq[u].y);
        *reinterpret_cast<uint64_t*>(d + 2 * kPitchQ) = both(nq[u].z);
        *reinterpret_cast<uint64_t*>(d + 3 * kPitchQ) = both(nq[u].w);
      }
    }
  };

  uint64_t acc[2][8] = {};
  if (s0 < s1) fetch(s0);
#pragma unroll 1
  for (int64_t s = s0; s < s1; s++) {
    __syncthreads();
    stage();
    __syncthreads();
    if (s + 1 < s1) fetch(s + 1);
    const float* qr = qs + wr * kPitchQ + wj * 16;
#pragma unroll 4
    for (int r = wr; r < KSTEP; r += kWR, qr += kWR * kPitchQ) {
      const float* pr = ps + r * kPitchP + (lane ^ Cfg::turn(r >> 2)) * 4;
      const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(pr);
      ulonglong2 b[4];
#pragma unroll
      for (int c = 0; c < 4; c++) b[c] = *reinterpret_cast<const ulonglong2*>(qr + 4 * c);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        acc[0][2 * c] = ptx::fma_f32x2(a.x, b[c].x, acc[0][2 * c]);
        acc[1][2 * c] = ptx::fma_f32x2(a.y, b[c].x, acc[1][2 * c]);
        acc[0][2 * c + 1] = ptx::fma_f32x2(a.x, b[c].y, acc[0][2 * c + 1]);
        acc[1][2 * c + 1] = ptx::fma_f32x2(a.y, b[c].y, acc[1][2 * c + 1]);
      }
    }
  }

  // the sums to shared memory, those of the warps with the same rows added up, then the cluster's
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 8; c++)
    *reinterpret_cast<ulonglong2*>(smem + (wr * kTJ + wj * 8 + c) * kTI + 4 * lane) = make_ulonglong2(acc[0][c], acc[1][c]);
  const int rows = static_cast<int>(p.J - j0 < kTJ ? p.J - j0 : kTJ);
  if constexpr (kWR > 1) {
    __syncthreads();
    for (int e = t; e < rows * kTI; e += kThreads) {
      float z = 0.0f;
#pragma unroll
      for (int w = 0; w < kWR; w++) z += smem[w * kTJ * kTI + e];
      smem[e] = z;
    }
  }
  ptx::cluster_sync();
  const uint32_t mine = ptx::smem_u32(smem);
  for (int e = static_cast<int>(part) * kThreads + t; e < rows * kTI; e += static_cast<int>(parts) * kThreads) {
    const int64_t j = j0 + e / kTI, i = i0 + e % kTI;
    if (i >= p.I) continue;
    float z = 0.0f;
    if (parts == 1) {
      z = smem[e];
    } else {
#pragma unroll 4
      for (uint32_t g = 0; g < parts; g++) {
        float w;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(ptx::mapa(mine + 4 * e, g)) : "memory");
        z += w;
      }
    }
    if (p.bias != nullptr) z += load_float<TVB_F32>(p.bias, i);
    if (p.preact != nullptr) store_float<TVB_F32>(p.preact, j * p.I + i, z);
    float y = act_value(z, p.activation);
    if (p.residual != nullptr) y += load_float<TVB_F32>(p.residual, j * p.residual_ld + i);
    store_float<TVB_F32>(p.out, j * p.I + i, y);
  }
  ptx::cluster_sync();  // no CTA's shared memory is released while another may read it
}

template <int WJ, int KSTEP, bool P_MN, bool Q_MN>
int simt_run(int device, cudaStream_t stream, const LinearProduct& p) {
  using Cfg = SimtCfg<WJ, KSTEP>;
  auto kernel = linear_simt_kernel<WJ, KSTEP, P_MN, Q_MN>;
  static bool configured[64] = {};
  if (!configured[device & 63]) {
    TVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
    configured[device & 63] = true;
  }
  const int64_t tiles_i = ceil_div(p.I, Cfg::kTI), tiles = tiles_i * ceil_div(p.J, Cfg::kTJ);
  // r in parts until two CTAs per SM have work, each at least four steps of it
  int parts = 1;
  while (parts < 8 && tiles * parts < 2ll * sm_count(device) && p.R >= static_cast<int64_t>(parts) * 2 * 4 * KSTEP) parts *= 2;
  if (tiles * parts >= (int64_t(1) << 31)) return fail("tvb_linear: too many output tiles");
  auto vec = [](const void* base, int64_t ld) { return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && ld % 4 == 0; };
  return launch_dependent_cluster("linear_simt", kernel, parts, dim3(static_cast<unsigned>(tiles * parts)), dim3(kThreads), Cfg::kSmem, stream, p,
                                  static_cast<uint32_t>(tiles_i), static_cast<int>(vec(p.p, P_MN ? p.p_sr : p.p_si)),
                                  static_cast<int>(vec(p.q, Q_MN ? p.q_sr : p.q_sj)));
}

template <bool P_MN, bool Q_MN>
int simt_shape(int device, cudaStream_t stream, const LinearProduct& p) {
  if (p.J <= 8) return simt_run<1, 64, P_MN, Q_MN>(device, stream, p);
  if (p.J <= 32) return simt_run<4, 32, P_MN, Q_MN>(device, stream, p);
  return simt_run<8, 16, P_MN, Q_MN>(device, stream, p);
}

}  // namespace

int linear_simt(int device, cudaStream_t stream, const LinearProduct& p) {
  if (p.p_mn) return p.q_mn ? simt_shape<true, true>(device, stream, p) : simt_shape<true, false>(device, stream, p);
  return simt_shape<false, false>(device, stream, p);
}

}  // namespace tvb
