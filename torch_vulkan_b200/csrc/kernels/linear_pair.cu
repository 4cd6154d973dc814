// The 16-bit products of linear.h on tcgen05 when the output is large: bound by the tensor pipe.
//
// A cluster of two CTAs (the two SMs of a TPC) walks output tiles of 256 rows (j) x BN columns (i), BN a multiple of 32 up to 256.
// Each CTA stages 128 rows of Q and BN / 2 rows of P per 64 values of r; one lane of CTA 0 issues tcgen05.mma.cta_group::2 for
// both, and each CTA's TMEM receives its own 128 rows of the tile, in two buffers, so that a tile is read back under the next
// tile's MMAs. BN is 256 unless narrower tiles put more pairs to work.
//
// A launch takes one product or two: the backward pass multiplies dz by w and by x at once. The tiles of the product with the
// longer r come first; pairs that get one tile of it less than others start on the second product meanwhile, and the rest of its
// tiles are dealt out in turn. The schedule is computed from the sizes alone (no counters in memory), so launches share nothing.
//   warps 0-7: epilogue (warp w reads TMEM lanes 32 (w % 4) ..., half w / 4 of the columns)
//   warp 8, one lane: TMA; warp 9, one lane of CTA 0: MMA. All mbarrier waits are bounded.
#include <cuda.h>

#include <mutex>

#include "../core/common.h"
#include "../core/tensormap.h"
#include "launch.h"
#include "linear.h"
#include "linear_epilogue.cuh"
#include "ptx_pair.cuh"

namespace tvb {
namespace {

constexpr int kTileJ = 256, kRowsQ = 128, kStepR = 64;
constexpr int kStageQ = kRowsQ * 128, kStageP = 128 * 128, kStage = kStageQ + kStageP, kStages = 6;
constexpr int kEpiWarps = 8, kProducer = 8, kMma = 9, kThreads = 320, kTmemCols = 512;
constexpr int kSmemBytes = kStages * kStage + 1024 + 256;
constexpr int kBand = 16;  // tile rows per band of the tile order

struct PairProduct {
  CUtensorMap map_q, map_p;
  const void* bias;
  const void* residual;
  void* out;
  void* preact;
  int64_t residual_ld;
  int I, J, blocks, tiles, tiles_i, tiles_j, bn, q_mn, p_mn, activation, vector_ok;
  uint32_t idesc, stage_bytes;
};

struct PairParams {
  PairProduct prod[2];
  int extra;        // tiles of product 1 that a pair with fewer tiles of product 0 takes first
  int light_first;  // which pairs come first when the rest of product 1 is dealt out
  int* status;
};

// Walks the tiles of one pair: its tiles of product 0, its share of product 1.
struct PairSchedule {
  int pair, pairs, tile, heavy, is_light, rank_among, stage_of;
  __device__ PairSchedule(const PairParams& p, int pair_, int pairs_) : pair(pair_), pairs(pairs_) {
    const int rest = p.prod[0].tiles % pairs;
    heavy = rest;                       // pairs 0 ... rest - 1 have one tile of product 0 more than the others
    is_light = rest != 0 && pair >= rest;
    rank_among = is_light ? pair - rest : pair;
    stage_of = 0;
    tile = pair;
  }
  // The next tile: which product, its index; false at the end.
  __device__ bool next(const PairParams& p, int& product, int& index) {
    if (stage_of == 0) {
      if (tile < p.prod[0].tiles) {
        product = 0;
        index = tile;
        tile += pairs;
        return true;
      }
      stage_of = 1;
      tile = rank_among;
    }
    product = 1;
    const int light = heavy != 0 ? pairs - heavy : 0, early = light * p.extra;
    if (stage_of == 1) {
      if (is_light && tile < early && tile < p.prod[1].tiles) {
        index = tile;
        tile += light;
        return true;
      }
      stage_of = 2;
      int order = pair;
      if (heavy != 0 && p.light_first) order = is_light ? rank_among : light + pair;
      tile = early + order;
    }
    if (tile >= p.prod[1].tiles) return false;
    index = tile;
    tile += pairs;
    return true;
  }
};

__device__ __forceinline__ void pair_tile_coords(const PairProduct& d, int tile, int& tj, int& ti) {
  const int per_band = kBand * d.tiles_i, b = tile / per_band, first = b * kBand;
  const int rows = d.tiles_j - first < kBand ? d.tiles_j - first : kBand;
  const int r = tile - b * per_band;
  tj = first + r % rows;
  ti = r / rows;
}

__device__ __forceinline__ void activate32(float (&v)[32], int act) {
  switch (act) {
    case TVB_ACT_RELU:
#pragma unroll
      for (int e = 0; e < 32; e++) v[e] = act_value<true>(v[e], TVB_ACT_RELU);
      break;
    case TVB_ACT_GELU:
#pragma unroll
      for (int e = 0; e < 32; e++) v[e] = act_value<true>(v[e], TVB_ACT_GELU);
      break;
    case TVB_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < 32; e++) v[e] = act_value<true>(v[e], TVB_ACT_GELU_TANH);
      break;
    case TVB_ACT_SILU:
#pragma unroll
      for (int e = 0; e < 32; e++) v[e] = act_value<true>(v[e], TVB_ACT_SILU);
      break;
    default: break;
  }
}

template <bool BF16>
__device__ __forceinline__ void add32(const void* src, int64_t at, float (&v)[32]) {  // (16-byte aligned)
  const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at);
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const uint4 x = s[q];
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float2 f = unpack16<BF16>(w[e]);
      v[q * 8 + 2 * e] += f.x;
      v[q * 8 + 2 * e + 1] += f.y;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ void put32(void* dst, int64_t at, const float (&v)[32]) {
  uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + at);
#pragma unroll
  for (int q = 0; q < 4; q++)
    d[q] = make_uint4(pack16<BF16>(v[q * 8], v[q * 8 + 1]), pack16<BF16>(v[q * 8 + 2], v[q * 8 + 3]),
                      pack16<BF16>(v[q * 8 + 4], v[q * 8 + 5]), pack16<BF16>(v[q * 8 + 6], v[q * 8 + 7]));
}

// 32 neighbouring sums of row j, from column i on.
template <bool BF16>
__device__ __forceinline__ void finish32(const PairProduct& d, int64_t j, int i, const uint32_t (&acc)[32]) {
  if (j >= d.J || i >= d.I) return;
  float v[32];
#pragma unroll
  for (int e = 0; e < 32; e++) v[e] = __uint_as_float(acc[e]);
  const int64_t o = j * d.I + i;
  if (d.vector_ok && i + 32 <= d.I) {
    if (d.bias != nullptr) add32<BF16>(d.bias, i, v);
    if (d.preact != nullptr) put32<BF16>(d.preact, o, v);
    activate32(v, d.activation);
    if (d.residual != nullptr) add32<BF16>(d.residual, j * d.residual_ld + i, v);
    put32<BF16>(d.out, o, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 32; e++)
    if (i + e < d.I) {
      if (d.bias != nullptr) v[e] += load16<BF16>(d.bias, i + e);
      if (d.preact != nullptr) store16<BF16>(d.preact, o + e, v[e]);
    }
  activate32(v, d.activation);
#pragma unroll
  for (int e = 0; e < 32; e++)
    if (i + e < d.I) {
      if (d.residual != nullptr) v[e] += load16<BF16>(d.residual, j * d.residual_ld + i + e);
      store16<BF16>(d.out, o + e, v[e]);
    }
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1) linear_pair_kernel(const __grid_constant__ PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - ptx::smem_u32(smem_raw));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + kStages * kStage);
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

  PairSchedule sched(p, pair, pairs);
  int which, tile;
  if (warp == kProducer) {
    if (lane == 0) {
      long long it = 0;
      bool ok = true;
      while (ok && sched.next(p, which, tile)) {
        const PairProduct& d = p.prod[which];
        int tj, ti;
        pair_tile_coords(d, tile, tj, ti);
        const int row_q = tj * kTileJ + static_cast<int>(rank) * kRowsQ, half = d.bn >> 1;
        const int row_p = ti * d.bn + static_cast<int>(rank) * half;
        const bool p_two = half > 64;  // (an MN-major operand comes in boxes of 64 columns)
        for (int kb = 0; kb < d.blocks; kb++, it++) {
          const int s = static_cast<int>(it % kStages);
          ok = ptx::mbar_wait(empty0 + 8 * s, static_cast<uint32_t>((it / kStages) & 1) ^ 1u, abort_flag);
          if (!ok) break;
          const uint32_t dst = base + s * kStage;
          if (rank == 0) ptx::mbar_expect_tx(full0 + 8 * s, 2 * d.stage_bytes);  // both CTAs' boxes of this stage
          const uint32_t bar = ptx::mapa(full0 + 8 * s, 0);
          const int r = kb * kStepR;
          if (d.q_mn) {
            ptx::tma_load_2d_pair(dst, &d.map_q, row_q, r, bar);
            ptx::tma_load_2d_pair(dst + 8192, &d.map_q, row_q + 64, r, bar);
          } else {
            ptx::tma_load_2d_pair(dst, &d.map_q, r, row_q, bar);
          }
          if (d.p_mn) {
            ptx::tma_load_2d_pair(dst + kStageQ, &d.map_p, row_p, r, bar);
            if (p_two) ptx::tma_load_2d_pair(dst + kStageQ + 8192, &d.map_p, row_p + 64, r, bar);
          } else {
            ptx::tma_load_2d_pair(dst + kStageQ, &d.map_p, r, row_p, bar);
          }
        }
      }
      if (rank == 0) {
        // no copy of either CTA may still be in flight when the pair's shared memory is released
        const long long first = it > kStages ? it - kStages : 0;
        for (long long j = first; j < it; j++) {
          volatile int never = 0;
          ptx::mbar_wait(full0 + 8 * static_cast<int>(j % kStages), static_cast<uint32_t>((j / kStages) & 1), &never);
        }
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (lane == 0 && rank == 0) {
      long long it = 0;
      int n = 0;
      bool ok = true;
      for (; ok && sched.next(p, which, tile); n++) {
        const PairProduct& d = p.prod[which];
        const int acc = n & 1;
        ok = ptx::mbar_wait(tempty0 + 8 * acc, static_cast<uint32_t>((n >> 1) & 1) ^ 1u, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * 256);
        const uint64_t step_q = d.q_mn ? 128 : 2, step_p = d.p_mn ? 128 : 2;
        for (int kb = 0; kb < d.blocks; kb++, it++) {
          const int s = static_cast<int>(it % kStages);
          ok = ptx::mbar_wait(full0 + 8 * s, static_cast<uint32_t>((it / kStages) & 1), abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t at = base + s * kStage;
          uint64_t qd = d.q_mn ? ptx::tc_smem_desc_sw128_mn(at) : ptx::tc_smem_desc_sw128(at);
          uint64_t pd = d.p_mn ? ptx::tc_smem_desc_sw128_mn(at + kStageQ) : ptx::tc_smem_desc_sw128(at + kStageQ);
#pragma unroll
          for (int j = 0; j < kStepR / 16; j++) {
            ptx::tc_mma_pair<2>(d_tmem, qd, pd, d.idesc, (kb | j) != 0 ? 1u : 0u);
            qd += step_q;
            pd += step_p;
          }
          ptx::tc_commit_pair(empty0 + 8 * s);  // frees the stage in both CTAs
        }
        if (ok) ptx::tc_commit_pair(tfull0 + 8 * acc);
      }
    }
    __syncwarp();
  } else {
    int n = 0;
    for (; sched.next(p, which, tile); n++) {
      const PairProduct& d = p.prod[which];
      int tj, ti;
      pair_tile_coords(d, tile, tj, ti);
      const int acc = n & 1;
      if (!ptx::mbar_wait(tfull0 + 8 * acc, static_cast<uint32_t>((n >> 1) & 1), abort_flag)) break;
      ptx::tc_fence_after();
      const int64_t row = static_cast<int64_t>(tj) * kTileJ + rank * kRowsQ + (warp & 3) * 32 + lane;
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + static_cast<uint32_t>(acc * 256);
#pragma unroll 1
      for (int c = (warp >> 2) * 32; c < d.bn; c += 64) {
        uint32_t r[32];
        ptx::tmem_ld_32x32(taddr + c, r);
        ptx::tmem_ld_wait();
        finish32<BF16>(d, row, ti * d.bn + c, r);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa(tempty0 + 8 * acc, 0));
    }
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
template <bool BF16>
int max_pairs(int device, int* out) {
  static std::mutex mutex;
  static int known[64] = {};
  std::lock_guard<std::mutex> lock(mutex);
  int& n = known[device & 63];
  if (n == 0) {
    auto kernel = linear_pair_kernel<BF16>;
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

int pair_product(const LinearProduct& lp, int bn, PairProduct* d) {
  const int half = bn / 2;
  if (operand_map(&d->map_q, lp.q, lp.dtype, lp.q_mn, lp.J, lp.R, lp.q_mn ? lp.q_sr : lp.q_sj, kRowsQ) != 0 ||
      operand_map(&d->map_p, lp.p, lp.dtype, lp.p_mn, lp.I, lp.R, lp.p_mn ? lp.p_sr : lp.p_si, half) != 0)
    return -1;
  d->bias = lp.bias;
  d->residual = lp.residual;
  d->out = lp.out;
  d->preact = lp.preact;
  d->residual_ld = lp.residual_ld;
  d->I = static_cast<int>(lp.I);
  d->J = static_cast<int>(lp.J);
  d->blocks = static_cast<int>(ceil_div(lp.R, kStepR));
  d->tiles_i = static_cast<int>(ceil_div(lp.I, bn));
  d->tiles_j = static_cast<int>(ceil_div(lp.J, kTileJ));
  TVB_REQUIRE(static_cast<int64_t>(d->tiles_i) * d->tiles_j < (int64_t(1) << 30), "tvb_linear: too many output tiles");
  d->tiles = d->tiles_i * d->tiles_j;
  d->bn = bn;
  d->q_mn = lp.q_mn;
  d->p_mn = lp.p_mn;
  d->activation = lp.activation;
  const uintptr_t all = reinterpret_cast<uintptr_t>(lp.out) | reinterpret_cast<uintptr_t>(lp.preact) | reinterpret_cast<uintptr_t>(lp.bias) |
                        reinterpret_cast<uintptr_t>(lp.residual);
  d->vector_ok = (all & 15u) == 0 && lp.I % 8 == 0 && (lp.residual == nullptr || lp.residual_ld % 8 == 0);
  const uint32_t fmt = lp.dtype == TVB_BF16 ? 1 : 0;
  d->idesc = ptx::tc_instr_desc(1, fmt, fmt, kTileJ, bn) | (lp.q_mn ? ptx::kTcAMajorMN : 0u) | (lp.p_mn ? ptx::kTcBMajorMN : 0u);
  d->stage_bytes = kStageQ + (lp.p_mn ? (half > 64 ? 16384 : 8192) : half * 128);
  return 0;
}

// Columns per tile for a product alone in its launch. A step of a tile costs its SM 128 rows of Q and bn / 2 of P from the L2,
// which is what paces it (7 rounds of 256 columns: 215 us; 7 of 224: 218; 9 of 192: 249), so narrower tiles pay only where
// they fill SMs that would have none.
int pair_columns(const LinearProduct& lp, int pairs) {
  int best = 256;
  int64_t best_cost = -1;
  for (int bn = 256; bn >= 128; bn -= 32) {
    const int64_t tiles = ceil_div(lp.I, bn) * ceil_div(lp.J, kTileJ);
    const int64_t cost = ceil_div(tiles, pairs) * (256 + bn);
    if (best_cost < 0 || cost * 10 < best_cost * 9) {
      best = bn;
      best_cost = cost;
    }
  }
  return best;
}

template <bool BF16>
int pair_run(int device, cudaStream_t stream, const LinearProduct* lp, int count) {
  int pairs = 0;
  if (max_pairs<BF16>(device, &pairs) != 0) return -1;
  PairParams p{};
  if (count == 2 && lp[0].R < lp[1].R) {
    const LinearProduct swapped[2] = {lp[1], lp[0]};
    return pair_run<BF16>(device, stream, swapped, 2);
  }
  for (int k = 0; k < count; k++)
    if (pair_product(lp[k], count == 1 ? pair_columns(lp[k], pairs) : 256, &p.prod[k]) != 0) return -1;
  pairs = std::min(pairs, p.prod[0].tiles + p.prod[1].tiles);
  if (count == 2 && p.prod[0].tiles % pairs != 0) {
    const int a = p.prod[0].blocks, b = p.prod[1].blocks;
    p.extra = (2 * a + b) / (2 * b);  // a / b, rounded
    p.light_first = p.extra * b < a;
  }
  if (status_word(device, &p.status) != 0) return -1;
  return launch_dependent_cluster("linear_pair", linear_pair_kernel<BF16>, 2, dim3(2 * static_cast<unsigned>(pairs)), dim3(kThreads), kSmemBytes,
                                  stream, p);
}

}  // namespace

int linear_pair(int device, cudaStream_t stream, const LinearProduct* lp, int count) {
  return lp[0].dtype == TVB_BF16 ? pair_run<true>(device, stream, lp, count) : pair_run<false>(device, stream, lp, count);
}

}  // namespace tvb
