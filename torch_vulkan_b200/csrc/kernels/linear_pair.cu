// The 16-bit products of linear.h on tcgen05 when the output is large: bound by the tensor pipe.
//
// A cluster of two CTAs (the two SMs of a TPC) walks output tiles of 256 rows (j) x 256 columns (i): per 64 values of r each CTA
// stages 128 rows of Q and 128 rows of P, 32 KB, six stages deep, and one lane of CTA 0 issues tcgen05.mma.cta_group::2 for both.
// Each CTA's TMEM receives its own 128 rows of the tile, in two buffers, so that a tile is read back under the next tile's
// multiplications. With a long r tiles have 512 rows, in two halves that share P: 48 KB per stage for twice the work, so a third
// less to move per multiplication; the halves' sums fill the TMEM, and a tile's read-back is not overlapped. Tiles that do not
// fill a round of pairs are cut into smaller ones (256 rows, 256 or 128 columns).
// Outputs leave through shared memory and TMA stores (a thread of the epilogue holds a row's 64 columns; stored from
// registers they are 32 scattered pieces per instruction, and the read-back took four times as long).
// A launch takes one product or two (256-row tiles): the backward pass multiplies dz by w and by x at once. Who makes which tile, and
// when, stands in linear_schedule.h.
//
// Measured (us per call, seconds-long runs, in which the GPU is held at its power limit): 2048 x 4096 x 14336 bfloat16 with gelu and its
// input saved 213 (1.13 PFLOP/s; the product alone 195); its gradients 434, of which the pass over dz takes 40 and both products
// 385 (1.25 PFLOP/s).
//   warps 0-7: epilogue (warp w reads TMEM lanes 32 (w % 4) ..., every second 32 columns)
//   warp 8, one lane: TMA; warp 9, one lane of CTA 0: MMA. All mbarrier waits are bounded.
#include <cuda.h>

#include <mutex>

#include "../core/common.h"
#include "../core/tensormap.h"
#include "launch.h"
#include "linear.h"
#include "linear_epilogue.cuh"
#include "linear_schedule.h"
#include "ptx_pair.cuh"

namespace tvb {
namespace {

constexpr int kRowsQ = 128, kStepR = 64;
constexpr int kBoxQ = kRowsQ * 128;  // bytes of one half's rows of Q in a stage
// HALVES: 2 for tiles of 512 rows, 1 for tiles of 256.
template <int HALVES>
struct PairCfg {
  static constexpr int kP = HALVES * kBoxQ;  // where P begins in a stage
  static constexpr int kStage = kP + 128 * 128;
  static constexpr int kStages = HALVES == 2 ? 4 : 6;
};
constexpr int kRing = 192 * 1024;
static_assert(PairCfg<1>::kStages * PairCfg<1>::kStage == kRing && PairCfg<2>::kStages * PairCfg<2>::kStage == kRing, "the ring's size");
constexpr int kEpiWarps = 8, kProducer = 8, kMma = 9, kThreads = 320, kTmemCols = 512;
constexpr int kOut = 32 * 128;  // a warp's outputs on their way out: 32 rows x 64 columns, 128-byte swizzle
constexpr int kSmemBytes = kRing + kEpiWarps * kOut + 1024 + 256;

struct PairProduct {
  CUtensorMap map_q, map_p;  // boxes of 64 values of r x 128 (Q) or 64 (P) rows, or 64 x 64 where r is not contiguous
  CUtensorMap map_out, map_preact;  // boxes of 64 columns x 32 rows (where vector_ok)
  const void* bias;
  const void* residual;
  void* out;
  void* preact;
  int64_t residual_ld;
  PairExtent extent;
  int q_mn, p_mn, activation, vector_ok, alone;
  uint32_t fmt;  // instruction descriptor without the columns
};

struct PairParams {
  PairProduct prod[2];
  PairPlan plan;
  int* status;
};

__device__ __forceinline__ void fetch32(const void* base, int64_t at, uint4 (&x)[4]) {
  const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
  for (int q = 0; q < 4; q++) x[q] = s[q];
}
template <bool BF16>
__device__ __forceinline__ void add32(const uint4 (&x)[4], uint64_t (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 4; q++) {
    v[4 * q] = ptx::add_f32x2(v[4 * q], unpack16<BF16>(x[q].x));
    v[4 * q + 1] = ptx::add_f32x2(v[4 * q + 1], unpack16<BF16>(x[q].y));
    v[4 * q + 2] = ptx::add_f32x2(v[4 * q + 2], unpack16<BF16>(x[q].z));
    v[4 * q + 3] = ptx::add_f32x2(v[4 * q + 3], unpack16<BF16>(x[q].w));
  }
}

__device__ __forceinline__ void load32(uint32_t taddr, uint64_t (&v)[16]) {
  uint32_t acc[32];
  ptx::tmem_ld_32x32(taddr, acc);
  ptx::tmem_ld_wait();
#pragma unroll
  for (int e = 0; e < 16; e++) v[e] = ptx::pack_f32x2(acc[2 * e], acc[2 * e + 1]);
}

// 32 neighbouring outputs as 16 words, and those words into a row of the warp's staging tile (columns 32 q ...).
template <bool BF16>
__device__ __forceinline__ void pack32(const uint64_t (&v)[16], uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 16; e++) w[e] = pack16<BF16>(v[e]);
}
__device__ __forceinline__ void stage32(uint32_t tile, int lane, int q, const uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 4; e++)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + lane * 128 + (((4 * q + e) ^ (lane & 7)) << 4)), "r"(w[4 * e]),
                 "r"(w[4 * e + 1]), "r"(w[4 * e + 2]), "r"(w[4 * e + 3])
                 : "memory");
}

// The warp's staging tile to rows `row` ... and columns `col` ... of a matrix (what lies outside of it is not written).
__device__ __forceinline__ void store_tile(const CUtensorMap* map, uint32_t tile, int lane, int col, int row) {
  ptx::fence_proxy_async();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(col), "r"(row), "r"(tile)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// The staging tile may be written again.
__device__ __forceinline__ void wait_tile(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}

// Two times 32 sums (columns i ... i + 63 of this lane's row j; the warp's rows begin at row0), read from TMEM at `taddr`.
template <bool BF16>
__device__ __forceinline__ void finish64(const PairProduct& d, uint32_t taddr, uint32_t tile, int lane, int row0, int i) {
  uint32_t y[2][16];
  const bool live = row0 + lane < d.extent.J;
#pragma unroll
  for (int q = 0; q < 2; q++) {
    uint32_t w[16];
    uint64_t v[16];
    const int at = i + 32 * q;
    const bool inside = at + 32 <= d.extent.I;  // (else the row's last columns: fewer than 32, a multiple of 8)
    const int64_t r = static_cast<int64_t>(row0 + lane) * d.residual_ld + at;
    uint4 bias[4], residual[4];  // (on their way while the TMEM is read)
    if (d.bias != nullptr && inside) fetch32(d.bias, at, bias);
    if (d.residual != nullptr && live && inside) fetch32(d.residual, r, residual);
    load32(taddr + 32 * q, v);
    if (d.bias != nullptr) {
      if (inside) add32<BF16>(bias, v);
      else add_singly<BF16>(d.bias, at, d.extent.I - at, v);
    }
    if (d.preact != nullptr) {
      pack32<BF16>(v, w);
      if (q == 0) wait_tile(lane);
      stage32(tile, lane, q, w);
    }
    activate_pairs(v, d.activation);
    if (d.residual != nullptr && live) {
      if (inside) add32<BF16>(residual, v);
      else add_singly<BF16>(d.residual, r, d.extent.I - at, v);
    }
    pack32<BF16>(v, y[q]);
  }
  if (d.preact != nullptr) store_tile(&d.map_preact, tile, lane, i, row0);
  wait_tile(lane);
  stage32(tile, lane, 0, y[0]);
  stage32(tile, lane, 1, y[1]);
  store_tile(&d.map_out, tile, lane, i, row0);
}

// The same for a product alone (the gradients): nothing between the sums and their rounding. With a short r the read-back is what
// takes the time, and few warps do it: no branches, both reads of the TMEM on their way at once.
template <bool BF16>
__device__ __forceinline__ void store64(const PairProduct& d, uint32_t taddr, uint32_t tile, int lane, int row0, int i) {
  uint32_t acc[2][32], y[2][16];
  ptx::tmem_ld_32x32(taddr, acc[0]);
  ptx::tmem_ld_32x32(taddr + 32, acc[1]);
  ptx::tmem_ld_wait();
#pragma unroll
  for (int q = 0; q < 2; q++)
#pragma unroll
    for (int e = 0; e < 16; e++) y[q][e] = pack16<BF16>(ptx::pack_f32x2(acc[q][2 * e], acc[q][2 * e + 1]));
  wait_tile(lane);
  stage32(tile, lane, 0, y[0]);
  stage32(tile, lane, 1, y[1]);
  store_tile(&d.map_out, tile, lane, i, row0);
}

// 32 neighbouring sums of row j, from column i on, where rows or operands do not begin on 16 bytes.
template <bool BF16>
__device__ __forceinline__ void finish32(const PairProduct& d, uint32_t taddr, int64_t j, int i) {
  uint64_t v[16];
  load32(taddr, v);
  if (j >= d.extent.J || i >= d.extent.I) return;
  const int count = d.extent.I - i;
  const int64_t o = j * d.extent.I + i;
  if (d.bias != nullptr) add_singly<BF16>(d.bias, i, count, v);
  if (d.preact != nullptr) store_singly<BF16>(d.preact, o, count, v);
  activate_pairs(v, d.activation);
  if (d.residual != nullptr) add_singly<BF16>(d.residual, j * d.residual_ld + i, count, v);
  store_singly<BF16>(d.out, o, count, v);
}

// The roles' inner loops are run by one thread each, whose own instructions are the pace of everything (a copy instruction that
// follows some hundred clocks of index arithmetic halves what the copies can move): a position in the ring is a counter and a
// phase that step along, addresses and descriptors are sums, and the operands' orders are compile-time constants.
template <int STAGES>
struct RingAt {
  uint32_t slot = 0, phase = 0, rounds = 0;
  __device__ __forceinline__ void step() {
    if (++slot == STAGES) {
      slot = 0;
      phase ^= 1u;
      rounds++;
    }
  }
};

// The boxes of one tile (both CTAs of the pair run this, each for its own rows; `bar`: the leader's barriers, `bytes`: both CTAs').
template <int HALVES, bool Q_MN, bool P_MN>
__device__ __forceinline__ bool load_tile(const PairProduct& d, const PairTile& t, uint32_t rank, RingAt<PairCfg<HALVES>::kStages>& at, uint32_t base, uint32_t full0,
                                          uint32_t empty0, uint32_t bar0, volatile int* abort_flag) {
  constexpr int kStage = PairCfg<HALVES>::kStage, kPAt = PairCfg<HALVES>::kP;
  const int row_q = t.row + static_cast<int>(rank) * kRowsQ, row_p = t.col + static_cast<int>(rank) * (t.cols >> 1);
  const bool two = HALVES == 2 && t.halves == 2, wide = t.cols == kTileI;
  const uint32_t bytes = 2u * ((two ? 2 : 1) * kBoxQ + (wide ? 2 : 1) * 8192);
  const int blocks = d.extent.blocks;
  int r = 0;
#pragma unroll 1
  for (int kb = 0; kb < blocks; kb++, r += kStepR, at.step()) {
    if (!ptx::mbar_wait(empty0 + 8 * at.slot, at.phase ^ 1u, abort_flag)) return false;
    const uint32_t dst = base + at.slot * kStage, bar = bar0 + 8 * at.slot;
    if (rank == 0) ptx::mbar_expect_tx(full0 + 8 * at.slot, bytes);
    if (Q_MN) {
      ptx::tma_load_2d_pair(dst, &d.map_q, row_q, r, bar);
      ptx::tma_load_2d_pair(dst + 8192, &d.map_q, row_q + 64, r, bar);
      if (two) {
        ptx::tma_load_2d_pair(dst + kBoxQ, &d.map_q, row_q + kHalfJ, r, bar);
        ptx::tma_load_2d_pair(dst + kBoxQ + 8192, &d.map_q, row_q + kHalfJ + 64, r, bar);
      }
    } else {
      ptx::tma_load_2d_pair(dst, &d.map_q, r, row_q, bar);
      if (two) ptx::tma_load_2d_pair(dst + kBoxQ, &d.map_q, r, row_q + kHalfJ, bar);
    }
    if (P_MN) {
      ptx::tma_load_2d_pair(dst + kPAt, &d.map_p, row_p, r, bar);
      if (wide) ptx::tma_load_2d_pair(dst + kPAt + 8192, &d.map_p, row_p + 64, r, bar);
    } else {
      ptx::tma_load_2d_pair(dst + kPAt, &d.map_p, r, row_p, bar);
      if (wide) ptx::tma_load_2d_pair(dst + kPAt + 8192, &d.map_p, r, row_p + 64, bar);
    }
  }
  return true;
}

// The multiplications of one tile; half 0 into the sums at `d0`, half 1 (where there is one) into those at `d1`.
template <int HALVES, bool Q_MN, bool P_MN>
__device__ __forceinline__ bool multiply_tile(const PairProduct& d, const PairTile& t, RingAt<PairCfg<HALVES>::kStages>& at, uint32_t base, uint32_t full0, uint32_t empty0,
                                              uint32_t d0, uint32_t d1, volatile int* abort_flag) {
  constexpr int kStage = PairCfg<HALVES>::kStage, kPAt = PairCfg<HALVES>::kP;
  constexpr uint64_t kQ = Q_MN ? 128 : 2, kP = P_MN ? 128 : 2;  // 16 values of r, in the descriptors' units
  const uint32_t idesc = d.fmt | (static_cast<uint32_t>(t.cols >> 3) << 17);
  const uint64_t q0 = Q_MN ? ptx::tc_smem_desc_sw128_mn(base) : ptx::tc_smem_desc_sw128(base);
  const uint64_t p0 = P_MN ? ptx::tc_smem_desc_sw128_mn(base + kPAt) : ptx::tc_smem_desc_sw128(base + kPAt);
  const bool two = HALVES == 2 && t.halves == 2;
  const int blocks = d.extent.blocks;
  uint32_t more = 0;  // (the first instruction of a tile overwrites the sums)
#pragma unroll 1
  for (int kb = 0; kb < blocks; kb++, at.step()) {
    if (!ptx::mbar_wait(full0 + 8 * at.slot, at.phase, abort_flag)) return false;
    ptx::tc_fence_after();
    const uint64_t qd = q0 + at.slot * (kStage >> 4), pd = p0 + at.slot * (kStage >> 4);
#pragma unroll
    for (int j = 0; j < kStepR / 16; j++) ptx::tc_mma_pair<2>(d0, qd + kQ * j, pd + kP * j, idesc, j == 0 ? more : 1u);
    if (two) {
#pragma unroll
      for (int j = 0; j < kStepR / 16; j++) ptx::tc_mma_pair<2>(d1, qd + (kBoxQ >> 4) + kQ * j, pd + kP * j, idesc, j == 0 ? more : 1u);
    }
    more = 1;
    ptx::tc_commit_pair(empty0 + 8 * at.slot);  // frees the stage in both CTAs
  }
  return true;
}

template <int HALVES, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) linear_pair_kernel(const __grid_constant__ PairParams p) {
  constexpr int kStages = PairCfg<HALVES>::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - ptx::smem_u32(smem_raw));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + kRing + kEpiWarps * kOut);
  const uint32_t full0 = ptx::smem_u32(bars), empty0 = full0 + 8 * kStages, tfull0 = empty0 + 8 * kStages, tempty0 = tfull0 + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();  // 0: the CTA that issues the MMAs
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; s++) {
      ptx::mbar_init(full0 + 8 * s, 1);
      ptx::mbar_init(empty0 + 8 * s, 1);
    }
    for (int a = 0; a < 2; a++) {
      ptx::mbar_init(tfull0 + 8 * a, 1);
      ptx::mbar_init(tempty0 + 8 * a, 2 * kEpiWarps);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMma) ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), kTmemCols);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();  // both CTAs' barriers exist before either signals the other's
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  PairSchedule<HALVES> sched(p.plan, p.prod[0].extent, pair, pairs);
  PairTile t;
  if (warp == kProducer) {
    if (lane == 0) {
      RingAt<kStages> at;
      const uint32_t bar0 = ptx::mapa(full0, 0);  // the leader's barriers, from either CTA
      bool ok = true;
      while (ok && sched.next(p.plan, p.prod[0].extent, p.prod[1].extent, t)) {
        const PairProduct& d = p.prod[t.product];
        ok = d.q_mn   ? load_tile<HALVES, true, true>(d, t, rank, at, base, full0, empty0, bar0, abort_flag)
             : d.p_mn ? load_tile<HALVES, false, true>(d, t, rank, at, base, full0, empty0, bar0, abort_flag)
                      : load_tile<HALVES, false, false>(d, t, rank, at, base, full0, empty0, bar0, abort_flag);
      }
      // no copy of either CTA may still be in flight when the pair's shared memory is released: wait for the last filling of
      // every slot (slots before at.slot were filled in this turn of the ring, the others in the turn before, if there was one)
      for (uint32_t s = 0; rank == 0 && s < kStages; s++) {
        volatile int never = 0;
        if (s < at.slot) ptx::mbar_wait(full0 + 8 * s, at.phase, &never);
        else if (at.rounds != 0) ptx::mbar_wait(full0 + 8 * s, at.phase ^ 1u, &never);
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (lane == 0 && rank == 0) {
      RingAt<kStages> at;
      uint32_t used0 = 0, used1 = 0;  // tiles (or halves) that each buffer of sums has held
      int turn = 0;
      bool ok = true;
      while (ok && sched.next(p.plan, p.prod[0].extent, p.prod[1].extent, t)) {
        const PairProduct& d = p.prod[t.product];
        const bool both = t.halves == 2;
        const int buffer = both ? 0 : turn;  // (a single half takes the buffers in turn)
        if (!both) turn ^= 1;
        // the epilogues of both CTAs have read what the buffers held
        ok = ptx::mbar_wait(tempty0 + 8 * buffer, ((buffer ? used1 : used0) & 1u) ^ 1u, abort_flag);
        if (buffer) used1++;
        else used0++;
        if (ok && both) ok = ptx::mbar_wait(tempty0 + 8, (used1++ & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t d0 = tmem_base + static_cast<uint32_t>(buffer * 256), d1 = tmem_base + 256;
        ok = d.q_mn   ? multiply_tile<HALVES, true, true>(d, t, at, base, full0, empty0, d0, d1, abort_flag)
             : d.p_mn ? multiply_tile<HALVES, false, true>(d, t, at, base, full0, empty0, d0, d1, abort_flag)
                      : multiply_tile<HALVES, false, false>(d, t, at, base, full0, empty0, d0, d1, abort_flag);
        if (ok) {
          ptx::tc_commit_pair(tfull0 + 8 * buffer);
          if (both) ptx::tc_commit_pair(tfull0 + 8);
        }
      }
    }
    __syncwarp();
  } else {
    uint32_t used0 = 0, used1 = 0;
    int turn = 0;
    bool ok = true;
    while (ok && sched.next(p.plan, p.prod[0].extent, p.prod[1].extent, t)) {
      const PairProduct& d = p.prod[t.product];
      for (int h = 0; h < t.halves; h++) {
        const int b = t.halves == 2 ? h : turn;
        ok = ptx::mbar_wait(tfull0 + 8 * b, (b ? used1 : used0) & 1u, abort_flag, ptx::kWaitLimitCycles + d.extent.blocks * 4096ll);
        if (b) used1++;
        else used0++;
        if (!ok) break;
        ptx::tc_fence_after();
        const int row0 = t.row + h * kHalfJ + static_cast<int>(rank) * kRowsQ + (warp & 3) * 32;
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + static_cast<uint32_t>(b * 256);
        const uint32_t tile = base + kRing + warp * kOut;
#pragma unroll 1
        for (int c = (warp >> 2) * 64; c < t.cols; c += 128) {
          if (row0 >= d.extent.J || t.col + c >= d.extent.I) break;  // (nothing of it is inside)
          if (d.alone) {
            store64<BF16>(d, taddr + c, tile, lane, row0, t.col + c);
          } else if (d.vector_ok) {
            finish64<BF16>(d, taddr + c, tile, lane, row0, t.col + c);
          } else {
#pragma unroll 1
            for (int q = 0; q < 64; q += 32) finish32<BF16>(d, taddr + c + q, row0 + lane, t.col + c + q);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa(tempty0 + 8 * b, 0));
      }
      if (t.halves == 1) turn ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the last stores have been made
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag != 0) atomicExch(p.status, 2);
  ptx::cluster_sync();  // neither CTA signals the other, or is read by the other's MMAs, from here on
  if (warp == kMma) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

int operand_map(CUtensorMap* map, const void* base, int dtype, bool mn, int64_t count, int64_t r, int64_t ld, int box) {
  const CUtensorMapDataType dt = dtype == TVB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return make_tensor_map_2d(map, base, dt, mn ? count : r, mn ? r : count, ld * 2, 64, mn ? kStepR : box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Pairs of CTAs that the device holds at once (asked of the runtime once per device).
template <int HALVES, bool BF16>
int max_pairs(int device, int* out) {
  static std::mutex mutex;
  static int known[64] = {};
  std::lock_guard<std::mutex> lock(mutex);
  int& n = known[device & 63];
  if (n == 0) {
    auto kernel = linear_pair_kernel<HALVES, BF16>;
    TVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2 * static_cast<unsigned>(sm_count(device) / 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    TVB_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
    TVB_REQUIRE(clusters >= 1, "tvb_linear: the device holds no pair of CTAs of the tile kernel");
    n = clusters;
  }
  *out = n;
  return 0;
}

template <int HALVES>
int pair_product(const LinearProduct& lp, PairProduct* d) {
  if (operand_map(&d->map_q, lp.q, lp.dtype, lp.q_mn, lp.J, lp.R, lp.q_mn ? lp.q_sr : lp.q_sj, kRowsQ) != 0 ||
      operand_map(&d->map_p, lp.p, lp.dtype, lp.p_mn, lp.I, lp.R, lp.p_mn ? lp.p_sr : lp.p_si, 64) != 0)
    return -1;
  d->bias = lp.bias;
  d->residual = lp.residual;
  d->out = lp.out;
  d->preact = lp.preact;
  d->residual_ld = lp.residual_ld;
  PairExtent& e = d->extent;
  e.I = static_cast<int>(lp.I);
  e.J = static_cast<int>(lp.J);
  e.blocks = static_cast<int>(ceil_div(lp.R, kStepR));
  e.tiles_i = static_cast<int>(ceil_div(lp.I, kTileI));
  e.tiles_j = static_cast<int>(ceil_div(lp.J, PairSchedule<HALVES>::kTileJ));
  TVB_REQUIRE(static_cast<int64_t>(e.tiles_i) * e.tiles_j < (int64_t(1) << 28), "tvb_linear: too many output tiles");
  e.tiles = e.tiles_i * e.tiles_j;
  d->q_mn = lp.q_mn;
  d->p_mn = lp.p_mn;
  d->activation = lp.activation;
  const uintptr_t all = reinterpret_cast<uintptr_t>(lp.out) | reinterpret_cast<uintptr_t>(lp.preact) | reinterpret_cast<uintptr_t>(lp.bias) |
                        reinterpret_cast<uintptr_t>(lp.residual);
  d->vector_ok = (all & 15u) == 0 && lp.I % 8 == 0 && (lp.residual == nullptr || lp.residual_ld % 8 == 0);
  d->alone = d->vector_ok && lp.activation == TVB_ACT_NONE && lp.bias == nullptr && lp.preact == nullptr && lp.residual == nullptr;
  if (d->vector_ok) {
    const CUtensorMapDataType dt = lp.dtype == TVB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (make_tensor_map_2d(&d->map_out, lp.out, dt, lp.I, lp.J, lp.I * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B) != 0) return -1;
    if (lp.preact != nullptr && make_tensor_map_2d(&d->map_preact, lp.preact, dt, lp.I, lp.J, lp.I * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B) != 0)
      return -1;
  }
  const uint32_t fmt = lp.dtype == TVB_BF16 ? 1 : 0;
  d->fmt = ptx::tc_instr_desc(1, fmt, fmt, kHalfJ, 0) | (lp.q_mn ? ptx::kTcAMajorMN : 0u) | (lp.p_mn ? ptx::kTcBMajorMN : 0u);
  return 0;
}

template <int HALVES, bool BF16>
int pair_run(int device, cudaStream_t stream, const LinearProduct* lp, int count) {
  int pairs = 0;
  if (max_pairs<HALVES, BF16>(device, &pairs) != 0) return -1;
  PairParams p{};
  const bool swap = count == 2 && lp[0].R < lp[1].R;  // the longer r first
  if (count == 2 && pair_product<HALVES>(lp[swap ? 1 : 0], &p.prod[0]) != 0) return -1;
  if (pair_product<HALVES>(lp[count == 2 && !swap ? 1 : 0], &p.prod[1]) != 0) return -1;
  pairs = plan_pairs<HALVES>(p.prod[0].extent, p.prod[1].extent, pairs, &p.plan);
  if (status_word(device, &p.status) != 0) return -1;
  return launch_dependent_cluster("linear_pair", linear_pair_kernel<HALVES, BF16>, 2, dim3(2 * static_cast<unsigned>(pairs)), dim3(kThreads), kSmemBytes,
                                  stream, p);
}

}  // namespace

int linear_pair(int device, cudaStream_t stream, const LinearProduct* lp, int count) {
  // Tiles of 512 rows for a long r, whose sums are read back seldom enough (us, 512 / 256 rows: 8192^3 811 / 850, dx of 2048 x 4096 x
  // 14336 with its 14336 values of r 185 / 199, y with 4096 208 / 198, dw with 2048 214 / 202, both gradients at once 395 / 383).
  const bool tall = count == 1 && lp[0].R >= 8192;
  if (tall) return lp[0].dtype == TVB_BF16 ? pair_run<2, true>(device, stream, lp, count) : pair_run<2, false>(device, stream, lp, count);
  return lp[0].dtype == TVB_BF16 ? pair_run<1, true>(device, stream, lp, count) : pair_run<1, false>(device, stream, lp, count);
}

}  // namespace tvb
