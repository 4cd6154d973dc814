// The 16-bit products of linear.h on tcgen05 when the output is small: few rows (decoding, short prompts), or gradients with few
// tiles. Bound by the bytes of P (the weights), by what the SMs can fetch from the L2, or by latency.
//
// One CTA multiplies a tile of 128 values of i (the MMA's 128 rows) by TN values of j (its columns; the rows of a decoding step
// are 16 of them or more), over a slice of r; S slices in a cluster share a tile. S is what makes a product of 32 tiles fill 148
// SMs. The CTAs leave their float32 sums in their own shared memory, and each adds up, in rank order, 1 / S of the tile's columns
// of all S through distributed shared memory: no scratch in global memory, no counters and no atomics, so a launch repeats
// its results bit for bit and launches share nothing.
// From TN = 64 on two CTAs (the SMs of a TPC) work as a pair on 256 values of i (tcgen05 cta_group::2): each stages its 128 rows
// of P and half of Q, so an SM fetches 32 KB per 64 values of r instead of 48 at TN = 256 (24 instead of 32 at 128).
//   warp 4, one lane: TMA (128-byte swizzle) into a ring of stages of 64 values of r
//   warp 5, one lane (of the pair's first CTA): tcgen05.mma, float32 sums in TMEM; the warp owns the TMEM
//   warps 0-3: TMEM -> shared memory; then all warps: sums, bias, activation, residual, store
// An operand may be contiguous along r (K-major) or along i / j (MN-major: the transposed reads of the backward pass).
// Up to TN = 128 the ring is kept under half of an SM's shared memory: two CTAs per SM, so that one streams while the other is
// in its prologue or epilogue.
//
// Measured (us per call): 1 x 4096 x 14336 bfloat16 with tanh-gelu 22.2 (117 MB of weights, 5.3 TB/s); 16 x 14336 x 4096 float16 with a
// residual 23.8; 200 x 4096 x 6144 bfloat16 with silu 19.7 (50 MB; the steps' pace through the L2); both gradients of 1000 x 1024 x
// 1000 float16 with silu 19.0 with the pass over dz (26.7 in two launches).
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "../core/common.h"
#include "../core/tensormap.h"
#include "launch.h"
#include "linear.h"
#include "linear_epilogue.cuh"
#include "ptx_pair.cuh"

namespace tvb {
namespace {

constexpr int kRows = 128, kStepR = 64, kThreads = 192, kProducer = 4, kMma = 5;

template <int TN>
struct SplitCfg {
  static constexpr bool kPair = TN >= 64;
  static constexpr int kTileI = kPair ? 2 * kRows : kRows;  // of the pair
  static constexpr int kRowsQ = kPair ? TN / 2 : TN;        // values of j that a CTA stages
  static constexpr int kStageP = kRows * 128, kStageQ = kRowsQ * 128, kStage = kStageP + kStageQ;
  static constexpr int kBudget = TN <= 128 ? 100 * 1024 : 200 * 1024;
  static constexpr int kStages = kBudget / kStage < 8 ? kBudget / kStage : 8;
  static constexpr int kCtasPerSm = TN <= 128 ? 2 : 1;
  static constexpr int kTmemCols = TN < 32 ? 32 : TN;
  static constexpr int kSmemBytes = kStages * kStage + 1024 + 256;
  static_assert(kRows * TN * 4 <= kStages * kStage, "the sums do not fit the ring");
};

struct SplitParams {
  CUtensorMap map_p, map_q;
  const void* bias;
  const void* residual;
  void* out;
  void* preact;
  int64_t residual_ld;
  int I, J, blocks, tiles_j, activation, vector_ok;
  uint32_t idesc, ctas;  // ctas: of this product
  int* status;
};

// The orders of the operands: r contiguous in both; i in P (dx); i in P and j in Q (dw); or two products in one launch, the
// first CTAs' as kDx and the others' as kDw.
enum Order { kForward, kDx, kDw, kDxDw };

template <int ORDER>
struct SplitArgs {
  SplitParams product[ORDER == kDxDw ? 2 : 1];
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {  // (from mapa)
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// How a warp finishes its columns of a tile. The sums of column j (of the tile) lie at `at` + j rows of shared memory in each of
// the `parts` CTAs of ranks first_rank, first_rank + rank_step, ...
struct Finish {
  uint32_t at, parts, first_rank, rank_step;
  int i;            // the lane's first output
  int64_t row0;     // row of the output that column 0 is
  uint64_t bias[2];
};

constexpr int kWarps = kThreads / 32;

// U columns, j, j + kWarps, ...: four neighbouring outputs of each. There are few warps here and every instruction waits for the
// one before it, so the U columns go through each step together, without branches between them (with a branch for each of four
// columns, a tile of 256 took 11 us to leave).
template <bool BF16, int ACT, int U>
__device__ __forceinline__ void finish_columns(const SplitParams& p, const Finish& f, int j) {
  uint64_t s[U][2] = {};
  auto add = [&](int u, const float4& v) {
    s[u][0] = ptx::add_f32x2(s[u][0], ptx::pack_f32x2(__float_as_uint(v.x), __float_as_uint(v.y)));
    s[u][1] = ptx::add_f32x2(s[u][1], ptx::pack_f32x2(__float_as_uint(v.z), __float_as_uint(v.w)));
  };
  const uint32_t mine = f.at + j * (kRows * 4);
  if (f.parts == 1) {  // (as an address of the cluster a CTA's own sums would take the trip all the same)
#pragma unroll
    for (int u = 0; u < U; u++) add(u, ld_shared_f4(mine + u * kWarps * (kRows * 4)));
  } else {
#pragma unroll 1
    for (uint32_t g0 = 0; g0 < f.parts; g0 += 4) {  // (four CTAs' sums asked for at a time)
      float4 v[4][U];
#pragma unroll
      for (uint32_t g = 0; g < 4; g++) {
        const bool there = g0 + g < f.parts;
        const uint32_t from = ptx::mapa(mine, f.first_rank + (there ? g0 + g : g0) * f.rank_step);
#pragma unroll
        for (int u = 0; u < U; u++) {
          v[g][u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (there) v[g][u] = ld_cluster_f4(from + u * kWarps * (kRows * 4));
        }
      }
#pragma unroll
      for (uint32_t g = 0; g < 4; g++)
#pragma unroll
        for (int u = 0; u < U; u++) add(u, v[g][u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    s[u][0] = ptx::add_f32x2(s[u][0], f.bias[0]);
    s[u][1] = ptx::add_f32x2(s[u][1], f.bias[1]);
  }
  const int64_t row = f.row0 + j, step = static_cast<int64_t>(kWarps) * p.I;
  const int64_t o = row * p.I + f.i;
  if (p.vector_ok) {  // (I a multiple of 4, every pointer and row on 8 bytes)
    auto put = [&](void* dst) {
      uint16_t* to = static_cast<uint16_t*>(dst) + o;
#pragma unroll
      for (int u = 0; u < U; u++, to += step) *reinterpret_cast<uint2*>(to) = make_uint2(pack16<BF16>(s[u][0]), pack16<BF16>(s[u][1]));
    };
    if (p.preact != nullptr) put(p.preact);
#pragma unroll
    for (int u = 0; u < U; u++) s[u][0] = act_pair<ACT>(s[u][0]), s[u][1] = act_pair<ACT>(s[u][1]);
    if (p.residual != nullptr) {
      const uint16_t* from = static_cast<const uint16_t*>(p.residual) + row * p.residual_ld + f.i;
      uint2 r[U];
#pragma unroll
      for (int u = 0; u < U; u++, from += kWarps * p.residual_ld) r[u] = *reinterpret_cast<const uint2*>(from);
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u][0] = ptx::add_f32x2(s[u][0], unpack16<BF16>(r[u].x));
        s[u][1] = ptx::add_f32x2(s[u][1], unpack16<BF16>(r[u].y));
      }
    }
    put(p.out);
    return;
  }
  const int count = p.I - f.i;
#pragma unroll 1
  for (int u = 0; u < U; u++) {
    uint64_t z[2] = {s[0][0], s[0][1]};
#pragma unroll
    for (int w = 1; w < U; w++)
      if (u == w) z[0] = s[w][0], z[1] = s[w][1];
    if (p.preact != nullptr) store_singly<BF16>(p.preact, o + u * step, count, z);
    z[0] = act_pair<ACT>(z[0]);
    z[1] = act_pair<ACT>(z[1]);
    if (p.residual != nullptr) add_singly<BF16>(p.residual, (row + u * kWarps) * p.residual_ld + f.i, count, z);
    store_singly<BF16>(p.out, o + u * step, count, z);
  }
}

template <bool BF16, int ACT>
__device__ __forceinline__ void finish_tile(const SplitParams& p, const Finish& f, int j, int end) {
  constexpr int kAtOnce = 4;
#pragma unroll 1
  for (; j + (kAtOnce - 1) * kWarps < end; j += kAtOnce * kWarps) finish_columns<BF16, ACT, kAtOnce>(p, f, j);
#pragma unroll 1
  for (; j + kWarps < end; j += 2 * kWarps) finish_columns<BF16, ACT, 2>(p, f, j);
  if (j < end) finish_columns<BF16, ACT, 1>(p, f, j);
}

// Where a CTA stands in its cluster and what it multiplies.
struct SplitWork {
  uint32_t base, full0, empty0, tfull, half, first;
  int i0, j0, kb0, kb1;
};

// (The two threads that run these set the pace of the whole kernel: no index arithmetic in their loops.)
template <int TN, bool P_MN, bool Q_MN>
__device__ __forceinline__ void load_slices(const SplitParams& p, const SplitWork& w, volatile int* abort_flag) {
  using Cfg = SplitCfg<TN>;
  constexpr bool kPair = Cfg::kPair;
  uint32_t slot = 0, phase = 0;
  int r = w.kb0 * kStepR;
  const int row_q = w.j0 + static_cast<int>(w.half) * Cfg::kRowsQ;
  const uint32_t bars0 = kPair ? ptx::mapa(w.full0, w.first) : w.full0;  // the barriers that count the boxes: the pair's first CTA's
  auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (kPair) ptx::tma_load_2d_pair(dst, map, x, y, bar);
    else ptx::tma_load_2d(dst, map, x, y, bar);
  };
#pragma unroll 1
  for (int kb = w.kb0; kb < w.kb1; kb++, r += kStepR) {
    const uint32_t dst = w.base + slot * Cfg::kStage, bar = bars0 + 8 * slot;
    if (!ptx::mbar_wait(w.empty0 + 8 * slot, phase ^ 1u, abort_flag)) break;
    if (w.half == 0) ptx::mbar_expect_tx(w.full0 + 8 * slot, (kPair ? 2 : 1) * Cfg::kStage);
    if (P_MN) {
#pragma unroll
      for (int c = 0; c < kRows / 64; c++) load(dst + c * 8192, &p.map_p, w.i0 + c * 64, r, bar);
    } else {
      load(dst, &p.map_p, r, w.i0, bar);
    }
    if (Q_MN) {
#pragma unroll
      for (int c = 0; c < Cfg::kRowsQ / 64; c++) load(dst + Cfg::kStageP + c * 8192, &p.map_q, row_q + c * 64, r, bar);
    } else {
      load(dst + Cfg::kStageP, &p.map_q, r, row_q, bar);
    }
    if (++slot == Cfg::kStages) {
      slot = 0;
      phase ^= 1u;
    }
  }
  // no copy may still be in flight when the ring is used for the sums or released: the last filling of every slot
  const int filled = (w.kb1 - w.kb0) < Cfg::kStages ? w.kb1 - w.kb0 : Cfg::kStages;
  for (int s = 0; w.half == 0 && s < filled; s++) {  // (a pair's second CTA stays until the sums are joined)
    volatile int never = 0;
    ptx::mbar_wait(w.full0 + 8 * s, s < static_cast<int>(slot) ? phase : phase ^ 1u, &never);
  }
}

template <int TN, bool P_MN, bool Q_MN>
__device__ __forceinline__ void multiply_slices(const SplitParams& p, const SplitWork& w, uint32_t tmem, volatile int* abort_flag) {
  using Cfg = SplitCfg<TN>;
  constexpr bool kPair = Cfg::kPair;
  constexpr uint64_t kP = P_MN ? 128 : 2, kQ = Q_MN ? 128 : 2;  // 16 values of r, in the descriptors' units
  const uint64_t p0 = P_MN ? ptx::tc_smem_desc_sw128_mn(w.base) : ptx::tc_smem_desc_sw128(w.base);
  const uint64_t q0 = Q_MN ? ptx::tc_smem_desc_sw128_mn(w.base + Cfg::kStageP) : ptx::tc_smem_desc_sw128(w.base + Cfg::kStageP);
  uint32_t slot = 0, phase = 0, more = 0;
  bool ok = w.kb1 > w.kb0;
#pragma unroll 1
  for (int kb = w.kb0; kb < w.kb1; kb++) {
    ok = ptx::mbar_wait(w.full0 + 8 * slot, phase, abort_flag);
    if (!ok) break;
    ptx::tc_fence_after();
    const uint64_t pd = p0 + slot * (Cfg::kStage >> 4), qd = q0 + slot * (Cfg::kStage >> 4);
#pragma unroll
    for (int j = 0; j < kStepR / 16; j++) {
      if (kPair) ptx::tc_mma_pair<2>(tmem, pd + kP * j, qd + kQ * j, p.idesc, j == 0 ? more : 1u);
      else ptx::tc_mma<2>(tmem, pd + kP * j, qd + kQ * j, p.idesc, j == 0 ? more : 1u);
    }
    more = 1;
    if (kPair) ptx::tc_commit_pair_at(w.empty0 + 8 * slot, w.first);  // (in both CTAs)
    else ptx::tc_commit(w.empty0 + 8 * slot);
    if (++slot == Cfg::kStages) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if (ok) {
    if (kPair) ptx::tc_commit_pair_at(w.tfull, w.first);
    else ptx::tc_commit(w.tfull);
  }
}

template <int TN, int ORDER, bool BF16>
__global__ void __launch_bounds__(kThreads, SplitCfg<TN>::kCtasPerSm) linear_split_kernel(const __grid_constant__ SplitArgs<ORDER> args) {
  using Cfg = SplitCfg<TN>;
  static_assert(ORDER < kDw || Cfg::kRowsQ >= 64, "an MN-major operand comes in columns of 64 values");
  constexpr bool kPair = Cfg::kPair;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - ptx::smem_u32(smem_raw));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + Cfg::kStages * Cfg::kStage);
  const uint32_t full0 = ptx::smem_u32(bars), empty0 = full0 + 8 * Cfg::kStages, tfull = empty0 + 8 * Cfg::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * Cfg::kStages + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  const uint32_t rank = ptx::cluster_ctarank();
  // half: which CTA of its pair this is; the pair's first CTA (rank `first`) issues its MMAs
  const uint32_t half = kPair ? rank & 1u : 0u, first = rank - half, part = kPair ? rank >> 1 : rank, parts = kPair ? ctas >> 1 : ctas;
  const bool second = ORDER == kDxDw && blockIdx.x >= args.product[0].ctas;  // (the same for a whole cluster)
  const SplitParams& p = args.product[second ? 1 : 0];
  const int tile = static_cast<int>((blockIdx.x - (second ? args.product[0].ctas : 0u)) / ctas);
  const int i0 = tile / p.tiles_j * Cfg::kTileI + static_cast<int>(half) * kRows, j0 = tile % p.tiles_j * TN;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.blocks) * part / parts);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.blocks) * (part + 1) / parts);
  const SplitWork work{base, full0, empty0, tfull, half, first, i0, j0, kb0, kb1};
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; s++) {
      ptx::mbar_init(full0 + 8 * s, 1);
      ptx::mbar_init(empty0 + 8 * s, 1);
    }
    ptx::mbar_init(tfull, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kProducer && lane == 0 && kb1 > kb0) {
    ptx::prefetch_tensormap(&p.map_p);
    ptx::prefetch_tensormap(&p.map_q);
  }
  if (warp == kMma) {
    if (kPair) ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), Cfg::kTmemCols);
    else ptx::tmem_alloc(ptx::smem_u32(tmem_slot), Cfg::kTmemCols);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (kPair) ptx::cluster_sync();  // both CTAs' barriers exist before either signals the other's
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  if (warp == kProducer) {
    if (lane == 0) {
      if constexpr (ORDER == kDxDw) {
        if (second) load_slices<TN, true, true>(p, work, abort_flag);
        else load_slices<TN, true, false>(p, work, abort_flag);
      } else {
        load_slices<TN, ORDER != kForward, ORDER == kDw>(p, work, abort_flag);
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (lane == 0 && half == 0) {
      if constexpr (ORDER == kDxDw) {
        if (second) multiply_slices<TN, true, true>(p, work, tmem, abort_flag);
        else multiply_slices<TN, true, false>(p, work, tmem, abort_flag);
      } else {
        multiply_slices<TN, ORDER != kForward, ORDER == kDw>(p, work, tmem, abort_flag);
      }
    }
    __syncwarp();
  } else {
    const bool empty = kb1 == kb0;  // no values of r here: sums of nothing
    // (the longest sum, 2^31 values in a cluster of eight, takes 2.6 seconds; a step takes some 500 clocks)
    const bool ok = empty || ptx::mbar_wait(tfull, 0, abort_flag, ptx::kWaitLimitCycles + static_cast<long long>(kb1 - kb0) * 4096);
    ptx::tc_fence_after();
    const uint32_t dst = base + (warp * 32 + lane) * 4;
    if (ok) {
      const uint32_t from = tmem + (static_cast<uint32_t>(warp * 32) << 16);
      if (empty) {
#pragma unroll 4
        for (int c = 0; c < TN; c++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + c * (kRows * 4)), "r"(0u) : "memory");
      } else if constexpr (TN == 16) {
        uint32_t r[16];
        ptx::tmem_ld_32x16(from, r);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + e * (kRows * 4)), "r"(r[e]) : "memory");
      } else {
        constexpr int kAtOnce = TN < 64 ? TN : 64;
#pragma unroll 1
        for (int c = 0; c < TN; c += kAtOnce) {
          uint32_t r[kAtOnce / 32][32];
#pragma unroll
          for (int h = 0; h < kAtOnce / 32; h++) ptx::tmem_ld_32x32(from + c + 32 * h, r[h]);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < kAtOnce / 32; h++)
#pragma unroll
            for (int e = 0; e < 32; e++)
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + (c + 32 * h + e) * (kRows * 4)), "r"(r[h][e]) : "memory");
        }
      }
    }
    ptx::tc_fence_before();
  }
  ptx::cluster_sync();  // every CTA's sums are in its shared memory
  if (warp == kMma) {
    ptx::tc_fence_after();
    if (kPair) ptx::tmem_dealloc_pair(tmem, Cfg::kTmemCols);
    else ptx::tmem_dealloc(tmem, Cfg::kTmemCols);
  }
  if (*abort_flag == 0) {
    const int c0 = TN * static_cast<int>(part) / static_cast<int>(parts), c1 = TN * (static_cast<int>(part) + 1) / static_cast<int>(parts);
    // a lane keeps its four values of i, a warp takes every sixth column
    Finish f;
    f.at = base + lane * 16;
    f.parts = parts;
    f.first_rank = kPair ? half : 0;
    f.rank_step = kPair ? 2 : 1;
    f.i = i0 + lane * 4;
    f.row0 = j0;
    const int j = c0 + warp, end = c1 < p.J - j0 ? c1 : p.J - j0;
    if (f.i < p.I) {
      f.bias[0] = f.bias[1] = 0;
      if (p.bias != nullptr) add_singly<BF16>(p.bias, f.i, p.I - f.i, f.bias);
      switch (p.activation) {
        case TVB_ACT_RELU: finish_tile<BF16, TVB_ACT_RELU>(p, f, j, end); break;
        case TVB_ACT_GELU: finish_tile<BF16, TVB_ACT_GELU>(p, f, j, end); break;
        case TVB_ACT_GELU_TANH: finish_tile<BF16, TVB_ACT_GELU_TANH>(p, f, j, end); break;
        case TVB_ACT_SILU: finish_tile<BF16, TVB_ACT_SILU>(p, f, j, end); break;
        default: finish_tile<BF16, TVB_ACT_NONE>(p, f, j, end); break;
      }
    }
  } else if (threadIdx.x == 0) {
    atomicExch(p.status, 2);
  }
  ptx::cluster_sync();  // no CTA's shared memory is released while another may read it
}

// A map over one operand: `inner` contiguous values, `outer` rows.
int operand_map(CUtensorMap* map, const void* base, int dtype, int64_t inner, int64_t outer, int64_t ld, int box_outer) {
  const CUtensorMapDataType dt = dtype == TVB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return make_tensor_map_2d(map, base, dt, inner, outer, ld * 2, 64, box_outer, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The kernel's parameters for one product; `parts` slices of r.
template <int TN>
int split_params(int device, const LinearProduct& lp, int parts, SplitParams* p) {
  using Cfg = SplitCfg<TN>;
  if (lp.R > 0) {  // (a product over nothing: no box is ever loaded)
    if (operand_map(&p->map_p, lp.p, lp.dtype, lp.p_mn ? lp.I : lp.R, lp.p_mn ? lp.R : lp.I, lp.p_mn ? lp.p_sr : lp.p_si, lp.p_mn ? kStepR : kRows) != 0 ||
        operand_map(&p->map_q, lp.q, lp.dtype, lp.q_mn ? lp.J : lp.R, lp.q_mn ? lp.R : lp.J, lp.q_mn ? lp.q_sr : lp.q_sj, lp.q_mn ? kStepR : Cfg::kRowsQ) != 0)
      return -1;
  }
  p->bias = lp.bias;
  p->residual = lp.residual;
  p->out = lp.out;
  p->preact = lp.preact;
  p->residual_ld = lp.residual_ld;
  p->I = static_cast<int>(lp.I);
  p->J = static_cast<int>(lp.J);
  p->blocks = static_cast<int>(ceil_div(lp.R, kStepR));
  p->tiles_j = static_cast<int>(ceil_div(lp.J, TN));
  p->activation = lp.activation;
  const uintptr_t all = reinterpret_cast<uintptr_t>(lp.out) | reinterpret_cast<uintptr_t>(lp.preact) | reinterpret_cast<uintptr_t>(lp.bias) |
                        reinterpret_cast<uintptr_t>(lp.residual);
  p->vector_ok = (all & 7u) == 0 && lp.I % 4 == 0 && (lp.residual == nullptr || lp.residual_ld % 4 == 0);
  const uint32_t fmt = lp.dtype == TVB_BF16 ? 1 : 0;
  p->idesc = ptx::tc_instr_desc(1, fmt, fmt, Cfg::kTileI, TN) | (lp.p_mn ? ptx::kTcAMajorMN : 0u) | (lp.q_mn ? ptx::kTcBMajorMN : 0u);
  const int64_t ctas = ceil_div(lp.I, Cfg::kTileI) * p->tiles_j * (Cfg::kPair ? 2 * parts : parts);
  if (ctas >= (int64_t(1) << 30)) return fail("tvb_linear: too many output tiles");
  p->ctas = static_cast<uint32_t>(ctas);
  return status_word(device, &p->status);
}

template <int TN, int ORDER, bool BF16>
int split_run(int device, cudaStream_t stream, const LinearProduct* lp, int parts) {
  using Cfg = SplitCfg<TN>;
  auto kernel = linear_split_kernel<TN, ORDER, BF16>;
  static bool configured[64] = {};
  if (!configured[device & 63]) {
    TVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
    configured[device & 63] = true;
  }
  SplitArgs<ORDER> args{};
  uint32_t grid = 0;
  for (int k = 0; k < (ORDER == kDxDw ? 2 : 1); k++) {
    if (split_params<TN>(device, lp[k], parts, &args.product[k]) != 0) return -1;
    grid += args.product[k].ctas;
  }
  return launch_dependent_cluster("linear_split", kernel, Cfg::kPair ? 2 * parts : parts, dim3(grid), dim3(kThreads), Cfg::kSmemBytes, stream, args);
}

template <int TN, bool BF16>
int split_orders(int device, cudaStream_t stream, const LinearProduct* lp, int count, int parts) {
  if (count == 1 && !lp->q_mn)
    return lp->p_mn ? split_run<TN, kDx, BF16>(device, stream, lp, parts) : split_run<TN, kForward, BF16>(device, stream, lp, parts);
  if constexpr (TN >= 128) {
    if (count == 1 && lp->p_mn) return split_run<TN, kDw, BF16>(device, stream, lp, parts);
    if (count == 2 && lp[0].p_mn && !lp[0].q_mn && lp[1].p_mn && lp[1].q_mn) return split_run<TN, kDxDw, BF16>(device, stream, lp, parts);
  }
  return fail("tvb_linear: no kernel for this order of the operands");
}

// Clusters of `size` (1, 2, 3, 4, 6, 8) CTAs that run at once, one or two CTAs per SM, as the runtime counts them on a B200: a
// cluster stays within a GPC, so the larger ones leave SMs idle.
int clusters_at_once(int size, int per_sm) {
  constexpr int kOne[9] = {0, 148, 74, 45, 33, 0, 22, 0, 15}, kTwo[9] = {0, 296, 148, 93, 71, 0, 45, 0, 33};
  return per_sm == 2 ? kTwo[size] : kOne[size];
}

// The shape of a launch: which TN and S, and whether the kernel of CTA pairs (linear_pair.cu) is faster. The rule is a model of
// the time in us, fitted to 1137 measurements of both kernels (1 to 2048 rows, matrices from 512 x 512 to 4096 x 14336, every TN
// and S): its choices are 1.2 % slower than the best of each shape on average, 25 % at worst (1000 x 512 x 2048). What it
// says: a step (64 values of r) takes longer as more SMs ask the L2 at once, and as two CTAs share an SM; a tile's way out takes
// its time by its columns, more when sums are joined; clusters of more than four CTAs start late; and clusters run in whole
// rounds of those that fit at once (200 x 14336 x 4096 bfloat16 in 16 clusters: of six CTAs 33 us, of four 43, of eight, of which
// 15 fit, 55). From 74 tiles of 256 x 256 on (one for every pair of SMs) the pairs' kernel is taken whatever the model says: there
// the GPU is bound by its power, and fetching less counts for more than in a short run (2048 x 4096 x 14336 with gelu: 215 us
// against 255).
struct Shape {
  int tn, parts;
  double us;
};

// `count` products in one launch share TN and S.
double split_cost(const LinearProduct* lp, int count, int tn, int parts) {
  const bool pair = tn >= 64;
  const int size = pair ? 2 * parts : parts, per_sm = tn <= 128 ? 2 : 1, fit = clusters_at_once(size, per_sm);
  double clusters = 0, work = 0, longest = 0;
  for (int k = 0; k < count; k++) {
    const double n = static_cast<double>(ceil_div(lp[k].I, pair ? 2 * kRows : kRows) * ceil_div(lp[k].J, tn));
    const double steps = static_cast<double>(ceil_div(ceil_div(lp[k].R, kStepR), parts));
    clusters += n;
    work += n * steps;
    longest = std::max(longest, steps);
  }
  const double rounds = std::max(1.0, std::ceil(clusters / fit)), load = std::min<double>(clusters, fit) * size / 148;
  const double alone = tn <= 32 ? 0.227 : tn == 64 ? 0.252 : tn == 128 ? 0.305 : 0.298;
  const double step = alone * (1 + 0.314 * std::min(1.0, load)) * (1 + 0.511 * std::max(0.0, std::min<double>(load, per_sm) - 1));
  double us = 3.6 + 0.00826 * tn + std::max(longest, work / clusters * rounds) * step + 4.32 * (rounds - 1);
  if (parts > 1) us += 0.379 + 0.00859 * tn / parts;
  if (size > 4) us += 0.868;
  return us;
}

int64_t pair_tiles(const LinearProduct& lp) { return ceil_div(lp.I, 256) * ceil_div(lp.J, 256); }

double pair_cost(const LinearProduct& lp) {  // (fewer tiles than pairs)
  return 0.95 + static_cast<double>(ceil_div(lp.R, kStepR)) * (0.393 + 0.0124 * static_cast<double>(pair_tiles(lp)) / 74) + 3.31;
}

Shape split_shape(const LinearProduct* lp, int count) {
  const int least = lp[count - 1].q_mn ? 128 : 16;
  int64_t rows = 0, blocks = 0;
  for (int k = 0; k < count; k++) {
    rows = std::max(rows, lp[k].J);
    blocks = std::max(blocks, ceil_div(lp[k].R, kStepR));
  }
  int fits = least;  // the smallest TN that holds the rows
  while (fits < 256 && fits < rows) fits *= 2;
  Shape best{fits, 1, split_cost(lp, count, fits, 1)};
  for (int tn = fits; tn >= least && tn * 4 >= fits && (tn * 8 >= rows || tn >= 128); tn /= 2)
    for (int parts : {1, 2, 3, 4, 6, 8}) {
      if (parts > 1 && (parts > blocks || (tn >= 64 && parts > 4))) break;
      const double us = split_cost(lp, count, tn, parts);
      if (us < 0.96 * best.us) best = Shape{tn, parts, us};  // (a finer split has to be worth it)
    }
  return best;
}

}  // namespace

bool linear_large(const LinearProduct& lp) {
  if (lp.R == 0 || lp.J <= 64) return false;
  return pair_tiles(lp) >= 74 || pair_cost(lp) < split_shape(&lp, 1).us;
}

int linear_split(int device, cudaStream_t stream, const LinearProduct* lp, int count) {
  const Shape s = split_shape(lp, count);
  const bool bf16 = lp->dtype == TVB_BF16;
  switch (s.tn) {
    case 16: return bf16 ? split_orders<16, true>(device, stream, lp, count, s.parts) : split_orders<16, false>(device, stream, lp, count, s.parts);
    case 32: return bf16 ? split_orders<32, true>(device, stream, lp, count, s.parts) : split_orders<32, false>(device, stream, lp, count, s.parts);
    case 64: return bf16 ? split_orders<64, true>(device, stream, lp, count, s.parts) : split_orders<64, false>(device, stream, lp, count, s.parts);
    case 128: return bf16 ? split_orders<128, true>(device, stream, lp, count, s.parts) : split_orders<128, false>(device, stream, lp, count, s.parts);
    default: return bf16 ? split_orders<256, true>(device, stream, lp, count, s.parts) : split_orders<256, false>(device, stream, lp, count, s.parts);
  }
}

}  // namespace tvb
