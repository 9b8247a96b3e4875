// Matrix products grouped by expert, bf16 in, fp32 sums, and their gradients. The
// rows of a T-row matrix lie in groups, rows offsets[e] .. offsets[e + 1] going
// with expert e's weights W[e] (K x N):
//
//   forward          Y[r]  = X[r] W[e]            (T x N)    gemm_grouped_bf16
//   input gradient   dX[r] = dY[r] W[e]^T         (T x K)    gemm_grouped_dx_bf16
//   weight gradient  dW[e] = X_e^T dY_e           (K x N)    gemm_grouped_dw_bf16
//
// Rows of no group keep what the output held; an empty group's dW is zeros.
//
// One persistent CTA per SM over tiles of 128 rows by BN columns, the roles and the
// ring of gemm_bf16: a TMA producer, a tcgen05.mma issuer, eight epilogue warps (forms
// for CTA pairs and for groups of a few rows follow). No operand is transposed in
// memory: the forward product reads W N-major (as it lies) and the input gradient reads
// the same memory K-major; the weight gradient reads both X and dY "MN-major", a token
// a row of 128 bytes. The groups start at any row, which TMA allows (only the inner
// coordinate is aligned). 8192 rows over 16 groups of 2048 x 4096: 119 us in a burst
// (1150 TFLOP/s of what is asked, 1280 with the padding of ragged groups), 145 in a long
// run under the power cap.
//
// The weight gradient's last K block holds rows of the next group (or past T): the
// issuer's warp zeroes them in shared memory in both operands, up to the next
// multiple of 16, and issues only the MMAs (K = 16) that hold rows of the group. So
// what other groups' rows hold, infinities or NaN, cannot reach the sums.
//
// Rows of a partial tile are loaded in boxes of 32 where groups are small, so that a
// group of two rows costs 4 KiB of A a K block, not 16.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "../mtl_internal.hpp"
#include "tc_groups.cuh"

namespace mtl {

enum { kFwd = 0, kDx = 1, kDw = 2 };
constexpr int kGrThreads = 320, kGrM = 128, kGrK = 64;

template <int BN>
struct GrCfg {
  static constexpr uint32_t kAStage = kGrM * kGrK * 2, kBStage = kGrK * BN * 2;
  static constexpr uint32_t kStageBytes = kAStage + kBStage;
  static constexpr int kStages = (int)(196608 / kStageBytes);
  static constexpr uint32_t kTmemCols = 2 * BN;  // two accumulators
};
struct GrShared {
  uint4 stage[8][32 * 4];  // per epilogue warp: 64 bytes of 32 output rows
  uint64_t full[8], empty[8], tfull[2], tempty[2], drain;
  uint32_t tmem;
  int abort;
  GroupTable groups;
};
template <int BN>
constexpr int gr_smem() {
  return GrCfg<BN>::kStages * (int)GrCfg<BN>::kStageBytes + (int)sizeof(GrShared) + 1024;
}

struct GrArgs {
  void* out;
  const int* offsets;
  int T, cols, depth;  // rows of the row matrices; columns of the output; contraction (forward, dX)
  int out_rows;        // rows of dW[e]
  int groups;
  int a_box;  // rows per TMA box of A (forward, dX)
  int vec;    // rows of the output start on 16 bytes
  int chunked_a, chunked_b;  // MN-major operands loaded one box a K block
  int stall;  // the CTA whose producer stops after one K block, see take_stall
};

__device__ int g_grouped_timeouts;

struct GrTile {
  int e, m0, n0, rows;  // rows: valid output rows from m0 on
  int row0, depth;      // forward, dX: first row of A; dW: the group's first row and its row count
  int64_t crow;
};
template <int FORM, int TM, int BN, bool DEEP>  // TM rows a tile
struct GrWalk {
  GroupWalk g;
  __device__ __forceinline__ GrTile find(const GrArgs& p, const GroupTable* groups, int t, int tiles_m, int tiles_n) {
    GrTile c;
    if (FORM == kDw) {
      const int per = tiles_m * tiles_n, in = t % per;
      c.e = DEEP ? groups->cum[t / per] : t / per;  // DEEP: as order_groups left them
      c.m0 = in % tiles_m * TM;
      c.n0 = in / tiles_m * BN;
      c.rows = p.out_rows - c.m0;
      c.row0 = groups->lo[c.e];
      c.depth = groups->hi[c.e] - c.row0;
      c.crow = (int64_t)c.e * p.out_rows + c.m0;
    } else {
      g.find(groups, t, tiles_n, TM, BN, &c.row0, &c.rows, &c.n0);
      c.e = g.e;
      c.m0 = 0;
      c.depth = p.depth;
      c.crow = c.row0;
    }
    c.rows = min(c.rows, TM);
    return c;
  }
};

// Terms an accumulator runs for. The tensor core drops what an addition shifts out of fp32
// instead of rounding it, so the error grows with the terms (1352 of them: 1.4e-6 of the
// result). Where an fp32 output is the sum of more than 768 terms (DEEP), sums of 768 are
// added in registers, rounded to the nearest, and the error stays at 0.8e-6 (1.0e-6 over a
// million terms). Tiles of a single run are not to pay for the
// registers that hold those sums: with both kinds of tile in one loop a weight gradient went
// from 115 to 138 us. Forward and for the input gradient the terms are the same in every
// tile, so these are kernels of their own (8192 rows over 16 groups forward in fp32 take 161
// us, and 157 to 161 in one accumulator). A weight gradient's terms are its group's rows,
// which only the device knows: there the groups of a single run come first (order_groups) and
// the others after them, in a loop of their own. In this order the first loop costs 1 % for
// the registers of the second (128 rows a group 114.6 -> 115.9 us), in the other one 7 %.
//
// A bf16 output is DEEP above 32768 terms: by the same growth a run is off by 3.4e-5 of the
// result, and 8 million terms in one accumulator would be by 8e-3, more than the rounding to
// bf16. It also keeps every wait for an accumulator far below the limit, which the sums of a
// billion terms in one would pass.
template <typename OUT>
constexpr int kRunTerms = sizeof(OUT) == 4 ? 768 : 32768;
template <typename OUT, bool DEEP>
constexpr int kRunBlocks = DEEP ? kRunTerms<OUT> / kGrK : 1 << 28;

// A DEEP weight gradient's groups, those of a single run first: cum[i] is the i-th of them,
// cum[kMaxGroups] how many these are. Every thread of the CTA calls this, after build_groups,
// whose sums of tiles a weight gradient does not need.
template <typename OUT>
__device__ __forceinline__ void order_groups(GroupTable* g, int groups) {
  if (threadIdx.x < 32) {
    const uint32_t below = (1u << threadIdx.x) - 1;
    auto is_short = [&](int e) { return e < groups && g->hi[e] - g->lo[e] <= kRunTerms<OUT>; };
    int shorts = 0;
    for (int base = 0; base < groups; base += 32) shorts += __popc(__ballot_sync(0xffffffffu, is_short(base + (int)threadIdx.x)));
    int at = 0, rest = shorts;  // where the next of either goes
    for (int base = 0; base < groups; base += 32) {
      const int e = base + (int)threadIdx.x;
      const bool one = is_short(e);
      const uint32_t s = __ballot_sync(0xffffffffu, one), l = __ballot_sync(0xffffffffu, e < groups && !one);
      if (e < groups) g->cum[one ? at + __popc(s & below) : rest + __popc(l & below)] = e;
      at += __popc(s);
      rest += __popc(l);
    }
    if (threadIdx.x == 0) g->cum[kMaxGroups] = shorts;
  }
  __syncthreads();
}

// acc += W columns of a row of tensor memory, of which those from `cols` on are not wanted.
template <int W>
__device__ __forceinline__ void tmem_add(uint32_t addr, int cols, float (&acc)[W]) {
#pragma unroll
  for (int v = 0; v < W; v += 16) {  // 32 at a time leave too few registers
    if (v >= cols) break;  // uniform in the warp
    uint32_t r[16];
    tmem_ld16(addr + (uint32_t)v, r);
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[v + k] += __uint_as_float(r[k]);
  }
}

// W columns of a row, or zeros.
template <int W>
__device__ __forceinline__ void tmem_ld_row(uint32_t addr, bool zero, uint32_t (&r)[W]) {
  constexpr int kPart = W < 32 ? W : 32;
  uint32_t part[W / kPart][kPart];
  if (zero) {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < W / kPart; ++i) {
    if constexpr (kPart == 32)
      tmem_ld32_nowait(addr + (uint32_t)(i * kPart), part[i]);
    else
      tmem_ld16_nowait(addr, part[i]);
  }
#pragma unroll
  for (int i = 0; i < W / kPart; ++i) {
    tmem_wait_ld(part[i]);
#pragma unroll
    for (int j = 0; j < kPart; ++j) r[i * kPart + j] = part[i][j];
  }
}

template <int FORM, int BN, typename OUT, bool DEEP>
__global__ void __launch_bounds__(kGrThreads, 1)
    gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GrArgs p) {
  using Cfg = GrCfg<BN>;
  constexpr int kStages = Cfg::kStages, kRun = kRunBlocks<OUT, DEEP>;
  constexpr uint32_t kIdesc = idesc_bf16_f32(kGrM, BN, FORM == kDw, FORM != kDx);
  extern __shared__ unsigned char gr_raw[];
  unsigned char* ring =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gr_raw) + 1023) & ~uintptr_t(1023));
  GrShared* sh = reinterpret_cast<GrShared*>(ring + kStages * Cfg::kStageBytes);
  volatile int* abort = &sh->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&sh->tfull[a]), 1);
      mbar_init(smem_u32(&sh->tempty[a]), 8);
    }
    mbar_init(smem_u32(&sh->drain), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)),
                 "r"(Cfg::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  build_groups(&sh->groups, p.offsets, p.groups, p.T, kGrM);
  if constexpr (FORM == kDw && DEEP) order_groups<OUT>(&sh->groups, p.groups);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;

  const int tiles_m = FORM == kDw ? (p.out_rows + kGrM - 1) / kGrM : 0, tiles_n = (p.cols + BN - 1) / BN;
  const int ntiles = FORM == kDw ? tiles_m * tiles_n * p.groups : sh->groups.cum[p.groups] * tiles_n;  // checked by the host
  GrWalk<FORM, kGrM, BN, DEEP> walk;

  if (warp == 0) {
    // ── TMA producer (the whole warp waits, one lane issues) ──
    {
      bool ok = true;
      int s = 0;
      uint32_t ph = 0;
      int64_t issued = 0;
      const bool stalls = (int)blockIdx.x == p.stall;
      for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
        const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
        // a chunked operand comes in one box, zeros past its edges; other boxes that would
        // lie wholly past the output's rows or columns are not loaded:
        // what stale shared memory they leave feeds outputs that are not stored
        const int a_boxes = FORM == kDw ? (p.chunked_a ? kGrM / 64 : (c.rows + 63) / 64) : (c.rows + p.a_box - 1) / p.a_box;
        const int b_boxes = FORM == kDx ? 1 : p.chunked_b ? BN / 64 : min(BN / 64, (p.cols - c.n0 + 63) / 64);
        const uint32_t bytes = (uint32_t)(a_boxes * (FORM == kDw ? kGrK * 128 : p.a_box * 128)) +
                               (FORM == kDx ? Cfg::kBStage : (uint32_t)(b_boxes * kGrK * 128));
        const int kblocks = (c.depth + kGrK - 1) / kGrK;
        const int last = stalls ? min(kblocks, 1) : kblocks;
        for (int kb = 0; kb < last; ++kb) {
          ok = wait_warp(smem_u32(&sh->empty[s]), ph ^ 1, abort, &g_grouped_timeouts);
          if (!ok) break;
          if (elect_one()) {
          const uint32_t fb = smem_u32(&sh->full[s]);
          mbar_expect_tx(fb, bytes);
          const uint32_t a_dst = smem_u32(ring) + (uint32_t)(s * Cfg::kStageBytes), b_dst = a_dst + Cfg::kAStage;
          if (FORM == kDw) {
            if (p.chunked_a)
              tma_load_4d(a_dst, &tmA, 0, c.row0 + kb * kGrK, c.m0 / 64, 0, fb);
            else
              for (int b = 0; b < a_boxes; ++b)
                tma_load_3d(a_dst + b * (kGrK * 128), &tmA, c.m0 + b * 64, c.row0 + kb * kGrK, 0, fb);
            if (p.chunked_b)
              tma_load_4d(b_dst, &tmB, 0, c.row0 + kb * kGrK, c.n0 / 64, 0, fb);
            else
              for (int b = 0; b < b_boxes; ++b)
                tma_load_3d(b_dst + b * (kGrK * 128), &tmB, c.n0 + b * 64, c.row0 + kb * kGrK, 0, fb);
          } else {
            for (int b = 0; b < a_boxes; ++b)
              tma_load_3d(a_dst + b * p.a_box * 128, &tmA, kb * kGrK, c.row0 + b * p.a_box, 0, fb);
            if (FORM == kDx) {
              tma_load_3d(b_dst, &tmB, kb * kGrK, c.n0, c.e, fb);
            } else if (p.chunked_b) {
              tma_load_4d(b_dst, &tmB, 0, kb * kGrK, c.n0 / 64, c.e, fb);
            } else {
              for (int b = 0; b < b_boxes; ++b)
                tma_load_3d(b_dst + b * (kGrK * 128), &tmB, c.n0 + b * 64, kb * kGrK, c.e, fb);
            }
          }
          }
          __syncwarp();
          ++issued;
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (stalls) ok = ok && issued == 0;
      }
      if (!ok && lane == 0)  // the loads in flight land before the CTA leaves
        for (int64_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
          drain_phase(smem_u32(&sh->full[i % kStages]), (uint32_t)(i / kStages) & 1);
    }
  } else if (warp == 1) {
    // ── MMA issuer (the whole warp waits; one lane issues) ──
    int s = 0, i = 0;
    uint32_t ph = 0;
    bool ok = true;
    // MN-major: 64-value chunks kGrK * 128 bytes apart, a K = 16 slice is 16 rows of 128
    // bytes; K-major: rows of 128 bytes, a slice is 32 bytes further along the swizzled row
    constexpr uint32_t kAStep = (FORM == kDw ? 2048 : 32) >> 4, kBStep = (FORM == kDx ? 32 : 2048) >> 4;
    const uint64_t a0 = smem_desc(smem_u32(ring), FORM == kDw ? kGrK * 128 : 16, 1024);
    const uint64_t b0 = smem_desc(smem_u32(ring) + Cfg::kAStage, FORM == kDx ? 16 : kGrK * 128, 1024);
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
      const int kblocks = (c.depth + kGrK - 1) / kGrK;
      if (kblocks == 0) continue;
      int a = 0, in = 0;
      for (int kb = 0; ok && kb < kblocks; ++kb) {
        const bool first = in == 0, last = ++in == kRun || kb + 1 == kblocks;  // of an accumulator's run
        if (last) in = 0;
        if (first) {
          a = i & 1;
          ok = wait_warp(smem_u32(&sh->tempty[a]), ((i >> 1) & 1) ^ 1, abort, &g_grouped_timeouts);
          ++i;
          if (!ok) break;
        }
        const uint32_t d = tmem + (uint32_t)(a * BN);
        ok = wait_warp(smem_u32(&sh->full[s]), ph, abort, &g_grouped_timeouts);
        if (!ok) break;
        int steps = kGrK / 16;
        if (FORM == kDw && c.depth - kb * kGrK < kGrK) {
          const int live = c.depth - kb * kGrK, end = (live + 15) / 16 * 16;
          steps = end / 16;
          const int chunks = (kGrM + BN) / 64, words = (end - live) * 8;  // 16-byte words a chunk
          unsigned char* stage = ring + s * Cfg::kStageBytes;
          for (int w = lane; w < chunks * words; w += 32)
            *reinterpret_cast<uint4*>(stage + (w / words) * (kGrK * 128) + live * 128 + (w % words) * 16) =
                make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t off = (uint64_t)(s * (Cfg::kStageBytes >> 4));
          auto mma = [&](int kk) { tc_mma(d, a0 + off + kk * kAStep, b0 + off + kk * kBStep, kIdesc, !first || kk != 0); };
          if (steps == kGrK / 16) {
#pragma unroll
            for (int kk = 0; kk < kGrK / 16; ++kk) mma(kk);
          } else {
            for (int kk = 0; kk < steps; ++kk) mma(kk);
          }
          tc_commit(smem_u32(&sh->empty[s]));
          if (last) tc_commit(smem_u32(&sh->tfull[a]));
        }
        __syncwarp();
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok) drain_mmas<false>(smem_u32(&sh->drain));
  } else {
    // ── epilogue: warps 2..9 read TMEM lanes 32 (warp % 4) .. +32, half of the columns each ──
    const int q = warp & 3, half = (warp - 2) / 4, row = q * 32;
    int i = 0, t = blockIdx.x;
    bool ok = true;
    if constexpr (FORM == kDw || !DEEP) {
      const int end = DEEP ? sh->groups.cum[kMaxGroups] * tiles_m * tiles_n : ntiles;
      for (; ok && t < end; t += gridDim.x) {
        const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
        const bool empty = c.depth == 0;
        const int a = i & 1;
        if (!empty) {
          ok = wait_warp(smem_u32(&sh->tfull[a]), (i >> 1) & 1, abort, &g_grouped_timeouts);
          if (!ok) break;
          tc_fence_after();
          ++i;
        }
        if (row < c.rows) {  // uniform in the warp
          OUT* out = static_cast<OUT*>(p.out) + (c.crow + row) * (int64_t)p.cols;
          const uint32_t tbase = tmem + ((uint32_t)row << 16) + (uint32_t)(a * BN);
          constexpr int kW = 64 / sizeof(OUT), kChunks = BN / 2 / kW;  // columns a chunk, chunks a half
#pragma unroll 1
          for (int ch = half * kChunks; ch < (half + 1) * kChunks; ++ch) {
            const int col = c.n0 + ch * kW;
            if (col >= p.cols) break;
            uint32_t r[kW];
            tmem_ld_row(tbase + ch * kW, empty, r);
            store_rows(sh->stage[warp - 2], lane, c.rows - row, out, p.cols, col, p.vec, reinterpret_cast<const float(&)[kW]>(r));
          }
        }
        if (!empty) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->tempty[a]));
        }
      }
    }
    if constexpr (DEEP) {
      // tiles of several runs: every run's sums into registers, which frees the accumulators
      // before the rows are stored
      for (; ok && t < ntiles; t += gridDim.x) {
        const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
        const int kblocks = (c.depth + kGrK - 1) / kGrK, from = c.n0 + half * (BN / 2);
        constexpr int kW = 64 / sizeof(OUT);  // columns a piece
        float acc[BN / 2];
#pragma unroll
        for (int v = 0; v < BN / 2; ++v) acc[v] = 0.0f;
        for (int left = kblocks; left > 0; left -= kRun, ++i) {
          const int a = i & 1;
          ok = wait_warp(smem_u32(&sh->tfull[a]), (i >> 1) & 1, abort, &g_grouped_timeouts);
          if (!ok) break;
          tc_fence_after();
          if (row < c.rows) tmem_add(tmem + ((uint32_t)row << 16) + (uint32_t)(a * BN + half * (BN / 2)), p.cols - from, acc);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->tempty[a]));
        }
        if (ok && row < c.rows) {  // uniform in the warp
          OUT* out = static_cast<OUT*>(p.out) + (c.crow + row) * (int64_t)p.cols;
#pragma unroll
          for (int v = 0; v < BN / 2; v += kW)
            if (from + v < p.cols)
              store_rows(sh->stage[warp - 2], lane, c.rows - row, out, p.cols, from + v, p.vec, reinterpret_cast<const float(&)[kW]>(acc[v]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kTmemCols) : "memory");
}

// ── groups of a few rows: a decode step ─────────────────────────────────────
// A tile above costs 128 rows of MMAs however few its group has; with two rows an
// expert the weights' read time hides them, but not their power. Here the weights are
// the MMA's M operand (256 columns of the output as two runs of 128) and NT rows of the
// group its N operand, so a K block costs a quarter of the MMAs or less and the sums lie
// transposed: a lane of tensor memory holds one column of the output, and a row's 32
// columns leave a warp as one run.
template <int NT>
struct SlimCfg {
  static constexpr uint32_t kWStage = 256 * kGrK * 2, kXStage = NT * kGrK * 2, kStageBytes = kWStage + kXStage;
  static constexpr int kStages = 196608 / (int)kStageBytes;  // 5, or 4 with 64 rows
  static constexpr uint32_t kTmemCols = 4 * NT < 32 ? 32 : 4 * NT;  // two accumulators of two runs
};
template <int NT>
constexpr int slim_smem() {
  return SlimCfg<NT>::kStages * (int)SlimCfg<NT>::kStageBytes + (int)sizeof(GrShared) + 1024;
}

template <int FORM, int NT, typename OUT>
__global__ void __launch_bounds__(kGrThreads, 1)
    gemm_grouped_slim_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const GrArgs p) {
  using Cfg = SlimCfg<NT>;
  constexpr int kStages = Cfg::kStages, BN = 256, kRun = kRunBlocks<OUT, sizeof(OUT) == 4>;
  constexpr uint32_t kIdesc = idesc_bf16_f32(128, NT, FORM != kDx, false);
  extern __shared__ unsigned char gr_raw[];
  unsigned char* ring =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gr_raw) + 1023) & ~uintptr_t(1023));
  GrShared* sh = reinterpret_cast<GrShared*>(ring + kStages * Cfg::kStageBytes);
  volatile int* abort = &sh->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&sh->tfull[a]), 1);
      mbar_init(smem_u32(&sh->tempty[a]), 8);
    }
    mbar_init(smem_u32(&sh->drain), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)),
                 "r"(Cfg::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  build_groups(&sh->groups, p.offsets, p.groups, p.T, NT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;

  const int tiles_n = (p.cols + BN - 1) / BN, ntiles = sh->groups.cum[p.groups] * tiles_n;
  const int kblocks = (p.depth + kGrK - 1) / kGrK;
  GroupWalk walk;
  int row0, rows, n0;

  if (warp == 0) {
    // ── TMA producer (the whole warp waits, one lane issues) ──
    int s = 0;
    uint32_t ph = 0;
    int64_t issued = 0;
    bool ok = true;
    const bool stalls = (int)blockIdx.x == p.stall;
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      walk.find(&sh->groups, t, tiles_n, NT, BN, &row0, &rows, &n0);
      const int w_boxes = FORM == kDx ? 1 : p.chunked_b ? 4 : min(4, (p.cols - n0 + 63) / 64);
      const uint32_t bytes = Cfg::kXStage + (FORM == kDx ? Cfg::kWStage : (uint32_t)(w_boxes * kGrK * 128));
      const int last = stalls ? min(kblocks, 1) : kblocks;
      for (int kb = 0; kb < last; ++kb) {
        ok = wait_warp(smem_u32(&sh->empty[s]), ph ^ 1, abort, &g_grouped_timeouts);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t fb = smem_u32(&sh->full[s]), w_dst = smem_u32(ring) + (uint32_t)(s * Cfg::kStageBytes);
          mbar_expect_tx(fb, bytes);
          if (FORM == kDx) {
            tma_load_3d(w_dst, &tmW, kb * kGrK, n0, walk.e, fb);
          } else if (p.chunked_b) {
            tma_load_4d(w_dst, &tmW, 0, kb * kGrK, n0 / 64, walk.e, fb);
          } else {
            for (int b = 0; b < w_boxes; ++b) tma_load_3d(w_dst + b * (kGrK * 128), &tmW, n0 + b * 64, kb * kGrK, walk.e, fb);
          }
          // rows behind the group's feed columns that are not stored
          tma_load_3d(w_dst + Cfg::kWStage, &tmX, kb * kGrK, row0, 0, fb);
        }
        __syncwarp();
        ++issued;
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (stalls) ok = ok && issued == 0;
    }
    if (!ok && lane == 0)  // the loads in flight land before the CTA leaves
      for (int64_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
        drain_phase(smem_u32(&sh->full[i % kStages]), (uint32_t)(i / kStages) & 1);
  } else if (warp == 1) {
    // ── MMA issuer ──
    int s = 0, i = 0;
    uint32_t ph = 0;
    bool ok = true;
    constexpr uint32_t kWStep = (FORM == kDx ? 32 : 2048) >> 4, kXStep = 32 >> 4, kWRun = Cfg::kWStage / 2 >> 4;
    const uint64_t w0 = smem_desc(smem_u32(ring), FORM == kDx ? 16 : kGrK * 128, 1024);
    const uint64_t x0 = smem_desc(smem_u32(ring) + Cfg::kWStage, 16, 1024);
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      int a = 0, in = 0;
      for (int kb = 0; ok && kb < kblocks; ++kb) {
        const bool first = in == 0, last = ++in == kRun || kb + 1 == kblocks;  // of an accumulator's run
        if (last) in = 0;
        if (first) {
          a = i & 1;
          ok = wait_warp(smem_u32(&sh->tempty[a]), ((i >> 1) & 1) ^ 1, abort, &g_grouped_timeouts);
          ++i;
          if (!ok) break;
        }
        const uint32_t d = tmem + (uint32_t)(a * 2 * NT);
        ok = wait_warp(smem_u32(&sh->full[s]), ph, abort, &g_grouped_timeouts);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t off = (uint64_t)(s * (Cfg::kStageBytes >> 4));
#pragma unroll
          for (int kk = 0; kk < kGrK / 16; ++kk)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              tc_mma(d + (uint32_t)(r * NT), w0 + off + r * kWRun + kk * kWStep, x0 + off + kk * kXStep, kIdesc, !first || kk != 0);
          tc_commit(smem_u32(&sh->empty[s]));
          if (last) tc_commit(smem_u32(&sh->tfull[a]));
        }
        __syncwarp();
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok) drain_mmas<false>(smem_u32(&sh->drain));
  } else {
    // ── epilogue: a warp has 32 columns of the output, run (warp - 2) / 4 ──
    const int q = warp & 3, run = (warp - 2) / 4;
    int i = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < ntiles; t += gridDim.x) {
      walk.find(&sh->groups, t, tiles_n, NT, BN, &row0, &rows, &n0);
      const int col = n0 + run * 128 + q * 32 + lane;
      OUT* out = static_cast<OUT*>(p.out) + (int64_t)row0 * p.cols + col;
      const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(run * NT);
      if constexpr (sizeof(OUT) == 4) {  // the sums of every run
        float acc[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) acc[c] = 0.0f;
        for (int kb = 0; kb < kblocks; kb += kRun, ++i) {
          const int a = i & 1;
          ok = wait_warp(smem_u32(&sh->tfull[a]), (i >> 1) & 1, abort, &g_grouped_timeouts);
          if (!ok) break;
          tc_fence_after();
          tmem_add(lanes + (uint32_t)(a * 2 * NT), rows, acc);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->tempty[a]));
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < NT; ++c)
          if (c < rows && col < p.cols) out[(int64_t)c * p.cols] = acc[c];
      } else {
        const int a = i & 1;
        if (!wait_warp(smem_u32(&sh->tfull[a]), (i >> 1) & 1, abort, &g_grouped_timeouts)) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < NT; c += 16) {
          if (c >= rows) break;
          uint32_t r[16];
          tmem_ld16(lanes + (uint32_t)(a * 2 * NT + c), r);
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (c + v < rows && col < p.cols) out[(int64_t)(c + v) * p.cols] = __float2bfloat16_rn(__uint_as_float(r[v]));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->tempty[a]));
        ++i;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kTmemCols) : "memory");
}

// ── the same on CTA pairs: 256 x 256 tiles ──────────────────────────────────
// A pair loads 32 KiB a K block and CTA where one CTA a tile loads 48, which is less
// traffic and, in a run held to its power, less of that; but a group's rows come in tiles
// of 256. The weight gradient, whose rows are not a group's, gains most: its K loop is as
// short as its groups while every tile leaves 128 to 256 KiB. A last K block with rows
// behind the group lands on a barrier of each CTA's own; the CTA zeroes those rows and
// then tells the even CTA, which issues the MMAs. Sustained, us, against one CTA a tile
// (2048 x 4096): weight gradient of 8192 rows in 16 groups 181 and 210 (fp32), 145 and 173
// (bf16; storing by TMA from two 4 KiB buffers a warp, with fewer stages for their room,
// 158); forward with 4 groups 116 and 123, 8 groups 126 and 131, 16 groups 148 and 144.
//
// Weight gradients of short groups are stores for the most part, and take one stage of the
// ring for rows leaving in pieces of 128 bytes instead of 64 (store_rows). Sustained, us,
// 128 and 64 bytes, 16 groups (half to one and a half times as long each), 2048 x 4096: 128
// rows a group 107 and 129 (fp32), 72 and 80 (bf16); 256 rows 130 and 147, 104 and 104; 384
// rows 165 and 170, 129 and 125; 512 rows 197 and 189, 156 and 148.
template <int PIECE>  // bytes of an output row a store
struct PairCfg {
  static constexpr uint32_t kAStage = 128 * kGrK * 2, kStageBytes = 2 * kAStage;
  static constexpr int kStages = PIECE == 128 ? 5 : 6, kBN = 256;
};
template <int PIECE>
struct PairShared {
  uint4 stage[8][32 * PIECE / 16];  // per epilogue warp: output rows on their way out
  // full, tempty: the even CTA's are used
  uint64_t full[6], empty[6], tail[6], tfull[2], tempty[2], drain;
  uint32_t tmem;
  int abort;
  GroupTable groups;
};
template <int PIECE>
constexpr int pair_smem() {
  return PairCfg<PIECE>::kStages * (int)PairCfg<PIECE>::kStageBytes + (int)sizeof(PairShared<PIECE>) + 1024;
}

template <int FORM, int PIECE, typename OUT, bool DEEP>
__global__ void __launch_bounds__(kGrThreads, 1)
    gemm_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GrArgs p) {
  using Cfg = PairCfg<PIECE>;
  constexpr int kStages = Cfg::kStages, BN = Cfg::kBN, kRun = kRunBlocks<OUT, DEEP>;
  constexpr uint32_t kIdesc = idesc_bf16_f32(256, BN, FORM == kDw, FORM != kDx);
  extern __shared__ unsigned char gr_raw[];
  unsigned char* ring =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gr_raw) + 1023) & ~uintptr_t(1023));
  auto* sh = reinterpret_cast<PairShared<PIECE>*>(ring + kStages * Cfg::kStageBytes);
  volatile int* abort = &sh->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = blockIdx.x & 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 2);
      mbar_init(smem_u32(&sh->empty[s]), 1);
      mbar_init(smem_u32(&sh->tail[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&sh->tfull[a]), 1);
      mbar_init(smem_u32(&sh->tempty[a]), 16);
    }
    mbar_init(smem_u32(&sh->drain), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  build_groups(&sh->groups, p.offsets, p.groups, p.T, 256);
  if constexpr (FORM == kDw && DEEP) order_groups<OUT>(&sh->groups, p.groups);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are there
  tc_fence_after();
  const uint32_t tmem = sh->tmem;

  const int tiles_m = FORM == kDw ? (p.out_rows + 255) / 256 : 0, tiles_n = (p.cols + BN - 1) / BN;
  const int ntiles = FORM == kDw ? tiles_m * tiles_n * p.groups : sh->groups.cum[p.groups] * tiles_n;
  const int t0 = blockIdx.x / 2, tstep = gridDim.x / 2;
  GrWalk<FORM, 256, BN, DEEP> walk;

  if (warp == 0) {
    // ── TMA producer: this CTA's 128 rows of A and 128 columns of B ──
    int s = 0;
    uint32_t ph = 0, tails = 0, tph = 0;  // stages that tail was used for, the parity of its last use: a bit a stage
    int64_t issued = 0;
    bool ok = true;
    const bool stalls = (int)blockIdx.x == p.stall;
    for (int t = t0; ok && t < ntiles; t += tstep) {
      const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
      const int m0 = c.m0 + rank * 128, n0 = c.n0 + rank * 128;
      const int rows = min(max(c.rows - rank * 128, 0), 128), cols = min(max(p.cols - n0, 0), 128);
      // boxes; what would lie wholly past the output's rows or columns is not loaded
      const int a_boxes = FORM == kDw ? (rows + 63) / 64 : (rows + p.a_box - 1) / p.a_box;
      const int b_boxes = FORM == kDx ? (cols > 0 ? 1 : 0) : (cols + 63) / 64;
      const bool a_one = FORM == kDw && p.chunked_a && a_boxes, b_one = FORM != kDx && p.chunked_b && b_boxes;
      const uint32_t a_bytes = FORM == kDw ? (uint32_t)((a_one ? 2 : a_boxes) * kGrK * 128) : (uint32_t)(a_boxes * p.a_box * 128);
      const uint32_t bytes = a_bytes + (FORM == kDx ? (uint32_t)b_boxes * Cfg::kAStage : (uint32_t)((b_one ? 2 : b_boxes) * kGrK * 128));
      const int kblocks = (c.depth + kGrK - 1) / kGrK;
      const int last = stalls ? min(kblocks, 1) : kblocks;
      for (int kb = 0; kb < last; ++kb) {
        ok = wait_warp(smem_u32(&sh->empty[s]), ph ^ 1, abort, &g_grouped_timeouts);
        if (!ok) break;
        if (elect_one()) {
          const bool tail = FORM == kDw && c.depth - kb * kGrK < kGrK;
          const uint32_t a_dst = smem_u32(ring) + (uint32_t)(s * Cfg::kStageBytes), b_dst = a_dst + Cfg::kAStage;
          const uint32_t fb = tail ? smem_u32(&sh->tail[s]) : map_rank(smem_u32(&sh->full[s]), 0);
          if (tail)
            mbar_expect_tx(fb, bytes);
          else
            mbar_expect_tx_cluster(fb, bytes);
          if (FORM == kDw) {
            const int row = c.row0 + kb * kGrK;
            if (a_one)
              tma_load_4d_pair(a_dst, &tmA, 0, row, m0 / 64, 0, fb);
            else
              for (int i = 0; i < a_boxes; ++i) tma_load_3d_pair(a_dst + i * (kGrK * 128), &tmA, m0 + i * 64, row, 0, fb);
            if (b_one)
              tma_load_4d_pair(b_dst, &tmB, 0, row, n0 / 64, 0, fb);
            else
              for (int i = 0; i < b_boxes; ++i) tma_load_3d_pair(b_dst + i * (kGrK * 128), &tmB, n0 + i * 64, row, 0, fb);
          } else {
            for (int i = 0; i < a_boxes; ++i)
              tma_load_3d_pair(a_dst + i * p.a_box * 128, &tmA, kb * kGrK, c.row0 + rank * 128 + i * p.a_box, 0, fb);
            if (FORM == kDx) {
              if (b_boxes) tma_load_3d_pair(b_dst, &tmB, kb * kGrK, n0, c.e, fb);
            } else if (b_one) {
              tma_load_4d_pair(b_dst, &tmB, 0, kb * kGrK, n0 / 64, c.e, fb);
            } else {
              for (int i = 0; i < b_boxes; ++i)
                tma_load_3d_pair(b_dst + i * (kGrK * 128), &tmB, n0 + i * 64, kb * kGrK, c.e, fb);
            }
          }
        }
        if (FORM == kDw && c.depth - kb * kGrK < kGrK) {
          tph = tails >> s & 1 ? tph ^ 1u << s : tph;
          tails |= 1u << s;
        }
        __syncwarp();
        ++issued;
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (stalls) ok = ok && issued == 0;
    }
    if (!ok && lane == 0) {  // the loads in flight land before the CTAs leave
      if (FORM == kDw)
        for (int i = 0; i < kStages; ++i)
          if (tails >> i & 1) drain_phase(smem_u32(&sh->tail[i]), tph >> i & 1);
      if (rank == 0) {
        for (int64_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
          drain_phase(smem_u32(&sh->full[i % kStages]), (uint32_t)(i / kStages) & 1);
      } else {  // its loads count on the even CTA's barriers, which it cannot wait on: many times what a load takes
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 1000000) __nanosleep(10000);
      }
    }
  } else if (warp == 1) {
    // ── MMA issuer (even CTA); both: a group's last K block made clean ──
    int s = 0, i = 0;
    uint32_t ph = 0, tph = 0;  // tph: a bit a stage
    bool ok = true;
    constexpr uint32_t kAStep = (FORM == kDw ? 2048 : 32) >> 4, kBStep = (FORM == kDx ? 32 : 2048) >> 4;
    const uint64_t a0 = smem_desc(smem_u32(ring), FORM == kDw ? kGrK * 128 : 16, 1024);
    const uint64_t b0 = smem_desc(smem_u32(ring) + Cfg::kAStage, FORM == kDx ? 16 : kGrK * 128, 1024);
    // rows `live` .. up to a multiple of 16 of the stage zeroed, then the even CTA told
    auto clean = [&](int st, int live) {
      const bool here = wait_warp(smem_u32(&sh->tail[st]), tph >> st & 1, abort, &g_grouped_timeouts);
      tph ^= 1u << st;
      if (!here) return false;
      const int end = (live + 15) / 16 * 16, words = (end - live) * 8;
      unsigned char* stage = ring + st * Cfg::kStageBytes;
      for (int w = lane; w < 4 * words; w += 32)
        *reinterpret_cast<uint4*>(stage + (w / words) * (kGrK * 128) + live * 128 + (w % words) * 16) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_release_cluster(map_rank(smem_u32(&sh->full[st]), 0));
      return true;
    };
    for (int t = t0; ok && t < ntiles; t += tstep) {
      const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
      const int kblocks = (c.depth + kGrK - 1) / kGrK, live = FORM == kDw ? c.depth % kGrK : 0;
      if (kblocks == 0) continue;
      if (rank == 1) {
        if (live) ok = clean((s + kblocks - 1) % kStages, live);
        s = (s + kblocks) % kStages;
        continue;
      }
      int a = 0, in = 0;
      for (int kb = 0; ok && kb < kblocks; ++kb) {
        const bool first = in == 0, last = ++in == kRun || kb + 1 == kblocks;  // of an accumulator's run
        if (last) in = 0;
        if (first) {
          a = i & 1;
          ok = wait_warp(smem_u32(&sh->tempty[a]), ((i >> 1) & 1) ^ 1, abort, &g_grouped_timeouts);
          ++i;
          if (!ok) break;
        }
        const uint32_t d = tmem + (uint32_t)(a * BN);
        int steps = kGrK / 16;
        if (live && kb + 1 == kblocks) {
          steps = (live + 15) / 16;
          ok = clean(s, live);
          if (!ok) break;
        }
        ok = wait_warp(smem_u32(&sh->full[s]), ph, abort, &g_grouped_timeouts);
        if (!ok) break;
        if (live && kb + 1 == kblocks) mbar_acquire_cluster(smem_u32(&sh->full[s]), ph);  // the odd CTA's zeros, see clean
        tc_fence_after();
        if (elect_one()) {
          const uint64_t off = (uint64_t)(s * (Cfg::kStageBytes >> 4));
          if (steps == kGrK / 16) {
#pragma unroll
            for (int kk = 0; kk < kGrK / 16; ++kk) tc_mma_pair(d, a0 + off + kk * kAStep, b0 + off + kk * kBStep, kIdesc, !first || kk != 0);
          } else {
            for (int kk = 0; kk < steps; ++kk) tc_mma_pair(d, a0 + off + kk * kAStep, b0 + off + kk * kBStep, kIdesc, !first || kk != 0);
          }
          tc_commit_pair(smem_u32(&sh->empty[s]));
          if (last) tc_commit_pair(smem_u32(&sh->tfull[a]));
        }
        __syncwarp();
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok && rank == 0) drain_mmas<true>(smem_u32(&sh->drain));
  } else {
    // ── epilogue: this CTA's 128 rows; a warp 32 of them, half of the columns ──
    const int q = warp & 3, half = (warp - 2) / 4, row = rank * 128 + q * 32;
    int i = 0, t = t0;
    bool ok = true;
    if constexpr (FORM == kDw || !DEEP) {
      const int end = DEEP ? sh->groups.cum[kMaxGroups] * tiles_m * tiles_n : ntiles;
      for (; ok && t < end; t += tstep) {
        const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
        const bool empty = c.depth == 0;
        const int a = i & 1;
        if (!empty) {
          ok = wait_warp(smem_u32(&sh->tfull[a]), (i >> 1) & 1, abort, &g_grouped_timeouts);
          if (!ok) break;
          tc_fence_after();
          ++i;
        }
        if (row < c.rows) {
          OUT* out = static_cast<OUT*>(p.out) + (c.crow + row) * (int64_t)p.cols;
          const uint32_t tbase = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * BN);
          constexpr int kW = PIECE / sizeof(OUT), kChunks = BN / 2 / kW;  // columns a chunk, chunks a half
#pragma unroll 1
          for (int ch = half * kChunks; ch < (half + 1) * kChunks; ++ch) {
            const int col = c.n0 + ch * kW;
            if (col >= p.cols) break;
            uint32_t r[kW];
            tmem_ld_row(tbase + ch * kW, empty, r);
            store_rows(sh->stage[warp - 2], lane, c.rows - row, out, p.cols, col, p.vec, reinterpret_cast<const float(&)[kW]>(r));
          }
        }
        if (!empty) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(&sh->tempty[a]), 0));
        }
      }
    }
    if constexpr (DEEP) {
      // tiles of several runs: every run's sums into registers, which frees the accumulators
      // before the rows are stored
      for (; ok && t < ntiles; t += tstep) {
        const GrTile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n);
        const int kblocks = (c.depth + kGrK - 1) / kGrK, from = c.n0 + half * (BN / 2);
        constexpr int kW = 64 / sizeof(OUT);  // columns a piece; 128 bytes spill registers
        float acc[BN / 2];
#pragma unroll
        for (int v = 0; v < BN / 2; ++v) acc[v] = 0.0f;
        for (int left = kblocks; left > 0; left -= kRun, ++i) {
          const int a = i & 1;
          ok = wait_warp(smem_u32(&sh->tfull[a]), (i >> 1) & 1, abort, &g_grouped_timeouts);
          if (!ok) break;
          tc_fence_after();
          if (row < c.rows) tmem_add(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * BN + half * (BN / 2)), p.cols - from, acc);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(&sh->tempty[a]), 0));
        }
        if (ok && row < c.rows) {  // uniform in the warp
          OUT* out = static_cast<OUT*>(p.out) + (c.crow + row) * (int64_t)p.cols;
#pragma unroll
          for (int v = 0; v < BN / 2; v += kW)
            if (from + v < p.cols)
              store_rows(sh->stage[warp - 2], lane, c.rows - row, out, p.cols, from + v, p.vec, reinterpret_cast<const float(&)[kW]>(acc[v]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other's loads, MMAs or arrivals may reach it
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ── host side ───────────────────────────────────────────────────────────────
static std::atomic<int> g_grouped_stalls{0};
void grouped_inject_stall(int launches) { g_grouped_stalls.store(launches > 0 ? launches : 0); }
cudaError_t grouped_set_wait_limit(unsigned long long ns) { return set_wait_limit_this_file(ns); }
int grouped_timeouts(bool reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_grouped_timeouts, sizeof v) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (reset && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_grouped_timeouts, &zero, sizeof zero);
  }
  return v;
}

// A row-major bf16 matrix of `cols` columns, a multiple of 64, as chunks of 64 columns:
// {64, rows, chunks, slices}. One box of box_rows x box_chunks chunks lies in shared
// memory as the MMA's MN-major operand does, so a K block is one TMA instruction
// instead of two to four (forward over 16 groups 138 -> 124 us).
static mtl_status make_chunk_map(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t slices,
                                 uint32_t box_rows, uint32_t box_chunks) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return fail(MTL_ERR_CUDA, "gemm_grouped: cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[4] = {64, rows, cols / 64, slices};
  cuuint64_t strides[3] = {cols * 2, 128, rows * cols * 2};
  cuuint32_t box[4] = {64, box_rows, box_chunks, 1}, estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MTL_ERR_ARGUMENT, "gemm_grouped: tensor map rejected (CUresult %d)", (int)r);
  return MTL_OK;
}

static const char* const kGrName[3] = {"gemm_grouped_bf16", "gemm_grouped_dx_bf16", "gemm_grouped_dw_bf16"};

// Arguments: out (B), two operands (B): X, W / dY, W / X, dY, offsets (B, i32, groups +
// 1), T, N, K, output type (i); ndrange = groups.
template <int FORM>
static mtl_status gr_check(const LaunchArgs& la, const uint64_t* bytes) {
  const char* who = kGrName[FORM];
  if (la.ndim != 1) return fail(MTL_ERR_ARGUMENT, "%s: ndrange must be one-dimensional (the group count)", who);
  const int64_t E = la.nd[0], T = la.a[4].i32, N = la.a[5].i32, K = la.a[6].i32;
  const int out = la.a[7].i32;
  if (T < 0 || N < 0 || K < 0) return fail(MTL_ERR_ARGUMENT, "%s: negative dimension", who);
  if (std::max({T, N, K}) > kMaxSize) return fail(MTL_ERR_UNSUPPORTED, "%s: a dimension above 2^31 - 256", who);
  if (N % 8 || K % 8)
    return fail(MTL_ERR_UNSUPPORTED, "%s: N and K must be multiples of 8 (16-byte rows), got N=%lld K=%lld", who, (long long)N,
                (long long)K);
  if (FORM != kDw && (FORM == kFwd ? K : N) == 0) return fail(MTL_ERR_ARGUMENT, "%s: the contraction must be positive", who);
  if (out != 0 && out != 1) return fail(MTL_ERR_ARGUMENT, "%s: the output type is 0 (fp32) or 1 (bf16), got %d", who, out);
  if (E > kMaxGroups) return fail(MTL_ERR_UNSUPPORTED, "%s: more than %d groups", who, kMaxGroups);
  const int wide = out ? 2 : 4;
  auto w = [&](int size) { return bytes_of({E, K, N, size}); };
  auto x = [&](int size) { return bytes_of({T, K, size}); };
  auto y = [&](int size) { return bytes_of({T, N, size}); };
  const uint64_t need[4] = {FORM == kFwd ? y(wide) : FORM == kDx ? x(wide) : w(wide), FORM == kDx ? y(2) : x(2),
                            FORM == kDw ? y(2) : w(2), bytes_of({E + 1, 4})};
  const char* what[3][4] = {{"Y", "X", "W", "the offsets"}, {"dX", "dY", "W", "the offsets"}, {"dW", "X", "dY", "the offsets"}};
  const unsigned align[4] = {out ? 1u : 3u, 15, 15, 3};
  for (int i = 0; i < 4; ++i) {
    if (!la.a[i].ptr && need[i]) return fail(MTL_ERR_ARGUMENT, "%s: %s must be a device buffer", who, what[FORM][i]);
    if (bytes[i] && bytes[i] < need[i])
      return fail(MTL_ERR_ARGUMENT, "%s: %s: %llu bytes, the launch touches %llu", who, what[FORM][i], (unsigned long long)bytes[i],
                  (unsigned long long)need[i]);
    if (la.a[i].ptr & align[i])
      return fail(MTL_ERR_ARGUMENT, "%s: %s must be %u-byte aligned", who, what[FORM][i], align[i] + 1);
  }
  const int64_t rows = FORM == kDw ? (K + 127) / 128 * E : (T + 127) / 128 + E, cols = FORM == kDx ? K : N;
  if ((FORM == kDw ? rows : (T + 31) / 32 + E) * ((cols + 127) / 128) > INT_MAX) return fail(MTL_ERR_UNSUPPORTED, "%s: more than 2^31 tiles", who);
  return MTL_OK;
}
mtl_status gemm_grouped_check(const LaunchArgs& la, const uint64_t* bytes) { return gr_check<kFwd>(la, bytes); }
mtl_status gemm_grouped_dx_check(const LaunchArgs& la, const uint64_t* bytes) { return gr_check<kDx>(la, bytes); }
mtl_status gemm_grouped_dw_check(const LaunchArgs& la, const uint64_t* bytes) { return gr_check<kDw>(la, bytes); }

template <int FORM, int BN, typename OUT, bool DEEP>
static cudaError_t gr_launch(const CUtensorMap& ta, const CUtensorMap& tb, const GrArgs& p, int64_t tiles,
                             const LaunchArgs& la, cudaStream_t s) {
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(gemm_grouped_kernel<FORM, BN, OUT, DEEP>, gr_smem<BN>(), la.device, &done);
  if (e != cudaSuccess) return e;
  const int grid = (int)std::min<int64_t>(tiles, la.sm_count);
  gemm_grouped_kernel<FORM, BN, OUT, DEEP><<<grid, kGrThreads, gr_smem<BN>(), s>>>(ta, tb, p);
  return cudaGetLastError();
}

template <int FORM, int NT, typename OUT>
static cudaError_t gr_launch_slim(const CUtensorMap& tx, const CUtensorMap& tw, const GrArgs& p, int64_t tiles,
                                  const LaunchArgs& la, cudaStream_t s) {
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(gemm_grouped_slim_kernel<FORM, NT, OUT>, slim_smem<NT>(), la.device, &done);
  if (e != cudaSuccess) return e;
  gemm_grouped_slim_kernel<FORM, NT, OUT><<<(int)std::min<int64_t>(tiles, la.sm_count), kGrThreads, slim_smem<NT>(), s>>>(tx, tw, p);
  return cudaGetLastError();
}

template <int FORM, int PIECE, typename OUT, bool DEEP>
static cudaError_t gr_launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const GrArgs& p, int64_t tiles,
                                  const LaunchArgs& la, cudaStream_t s) {
  auto kernel = gemm_grouped_pair_kernel<FORM, PIECE, OUT, DEEP>;
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(kernel, pair_smem<PIECE>(), la.device, &done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, la.sm_count / 2)));
  cfg.blockDim = dim3(kGrThreads);
  cfg.dynamicSmemBytes = pair_smem<PIECE>();
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, ta, tb, p);
}

template <int FORM, int BN>
static cudaError_t gr_launch_by(bool bf16, bool deep, const CUtensorMap& ta, const CUtensorMap& tb, const GrArgs& p, int64_t tiles,
                                const LaunchArgs& la, cudaStream_t s) {
  if (bf16)
    return deep ? gr_launch<FORM, BN, __nv_bfloat16, true>(ta, tb, p, tiles, la, s) : gr_launch<FORM, BN, __nv_bfloat16, false>(ta, tb, p, tiles, la, s);
  return deep ? gr_launch<FORM, BN, float, true>(ta, tb, p, tiles, la, s) : gr_launch<FORM, BN, float, false>(ta, tb, p, tiles, la, s);
}
template <int FORM, int PIECE>
static cudaError_t gr_launch_pair_by(bool bf16, bool deep, const CUtensorMap& ta, const CUtensorMap& tb, const GrArgs& p, int64_t tiles,
                                     const LaunchArgs& la, cudaStream_t s) {
  if (bf16)
    return deep ? gr_launch_pair<FORM, PIECE, __nv_bfloat16, true>(ta, tb, p, tiles, la, s)
                : gr_launch_pair<FORM, PIECE, __nv_bfloat16, false>(ta, tb, p, tiles, la, s);
  return deep ? gr_launch_pair<FORM, PIECE, float, true>(ta, tb, p, tiles, la, s) : gr_launch_pair<FORM, PIECE, float, false>(ta, tb, p, tiles, la, s);
}

template <int FORM>
static mtl_status gr_run(const LaunchArgs& la, cudaStream_t s) {
  const char* who = kGrName[FORM];
  const int T = la.a[4].i32, N = la.a[5].i32, K = la.a[6].i32, out = la.a[7].i32;
  const int E = (int)la.nd[0];
  const int cols = FORM == kDx ? K : N;
  if (E == 0 || cols == 0 || (FORM == kDw ? K : T) == 0) return MTL_OK;
  if (FORM == kDw && T == 0) {  // every group is empty
    cudaError_t e = cudaMemsetAsync(reinterpret_cast<void*>(la.a[0].ptr), 0, (size_t)E * K * N * (out ? 2 : 4), s);
    return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  }
  GrArgs p = {};
  p.out = reinterpret_cast<void*>(la.a[0].ptr);
  p.offsets = reinterpret_cast<const int*>(la.a[3].ptr);
  p.T = T;
  p.cols = cols;
  p.depth = FORM == kFwd ? K : N;
  p.out_rows = K;
  p.groups = E;
  p.stall = take_stall(g_grouped_stalls);
  p.vec = la.a[0].ptr % 16 == 0;  // N and K are multiples of 8
  // Pairs where their 256-row tiles waste little (groups of 768 rows on average) and
  // there is a tile for each.
  const int64_t col_tiles = (cols + 255) / 256, pair_tiles = (FORM == kDw ? (int64_t)E * ((K + 255) / 256) : T / 256) * col_tiles;
  // a group has T rows at most
  const bool deep = (FORM == kDw ? T : p.depth) > (out ? kRunTerms<__nv_bfloat16> : kRunTerms<float>);
  const bool pair = pair_tiles >= la.sm_count / 2 && (FORM == kDw || T >= 768 * (int64_t)E);
  // Rows of a group in the MMA's N operand, 32 or 64 of them, while a group has up to 16
  // or 40 on average and there are tiles for most SMs. Sustained, us, against tiles of 128
  // rows: 2 rows a group (32 groups, 2048 x 4096) 81.7 and 89.5, 8 rows 83.1 and 90.8, 32
  // rows (16 groups, 2048 x 2048) 25.5 with 64, 29.7 with 32 and 28.0, 64 rows 55 and 51.3.
  const int64_t slim_tiles = (int64_t)E * col_tiles;
  const int slim = FORM == kDw || (out && deep) || slim_tiles * 4 < la.sm_count * 3 || T > 40 * (int64_t)E ? 0 : T <= 16 * (int64_t)E ? 32 : 64;
  p.a_box = slim ? slim : T / E >= kGrM ? kGrM : 32;
  const void *A = reinterpret_cast<const void*>(la.a[1].ptr), *B = reinterpret_cast<const void*>(la.a[2].ptr);
  const int64_t row_tiles = FORM == kDw ? (int64_t)E * ((K + 127) / 128) : std::max<int64_t>(E, (T + 127) / 128);
  // always so for a weight gradient: without a pair tile for every two SMs it has less than one of 128 rows for each
  const bool narrow = !pair && !slim && row_tiles * col_tiles < la.sm_count;
  const int bn = narrow ? 128 : 256, box_n = pair ? 128 : bn;  // columns of B a tile, a box
  p.chunked_a = FORM == kDw && K % 64 == 0;
  p.chunked_b = FORM != kDx && N % 64 == 0;
  CUtensorMap ta, tb;
  mtl_status st = p.chunked_a ? make_chunk_map(&ta, A, K, T, 1, kGrK, kGrM / 64)
                              : make_bf16_map(&ta, A, FORM == kDx ? N : K, T, 1, FORM == kDw ? kGrK : p.a_box);
  if (st) return st;
  st = p.chunked_b ? make_chunk_map(&tb, B, N, FORM == kDw ? T : K, FORM == kDw ? 1 : E, kGrK, box_n / 64)
       : FORM == kDw ? make_bf16_map(&tb, B, N, T, 1, kGrK)
                     : make_bf16_map(&tb, B, N, K, E, FORM == kDx ? box_n : kGrK);
  if (st) return st;
  const int64_t tile_m = pair ? 256 : 128;
  const int64_t tiles = (FORM == kDw ? (int64_t)E * ((K + tile_m - 1) / tile_m) : T / tile_m + E) * ((cols + bn - 1) / bn);
  cudaError_t e;
  if (slim) {
    if constexpr (FORM != kDw) {
      const int64_t n = ((int64_t)T / slim + E) * col_tiles;
      if (slim == 32)
        e = out ? gr_launch_slim<FORM, 32, __nv_bfloat16>(ta, tb, p, n, la, s) : gr_launch_slim<FORM, 32, float>(ta, tb, p, n, la, s);
      else
        e = out ? gr_launch_slim<FORM, 64, __nv_bfloat16>(ta, tb, p, n, la, s) : gr_launch_slim<FORM, 64, float>(ta, tb, p, n, la, s);
    } else {
      e = cudaErrorInvalidValue;
    }
  } else if (pair && FORM == kDw && T <= (out ? 256 : 448) * (int64_t)E) {
    constexpr int kPiece = FORM == kDw ? 128 : 64;
    e = gr_launch_pair_by<FORM, kPiece>(out, deep, ta, tb, p, tiles, la, s);
  } else if (pair) {
    e = gr_launch_pair_by<FORM, 64>(out, deep, ta, tb, p, tiles, la, s);
  } else if (narrow) {
    e = gr_launch_by<FORM, 128>(out, deep, ta, tb, p, tiles, la, s);
  } else {
    if constexpr (FORM != kDw)
      e = gr_launch_by<FORM, 256>(out, deep, ta, tb, p, tiles, la, s);
    else
      e = cudaErrorInvalidValue;
  }
  return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}
mtl_status gemm_grouped_run(const LaunchArgs& la, void*, uint64_t, void* stream) { return gr_run<kFwd>(la, (cudaStream_t)stream); }
mtl_status gemm_grouped_dx_run(const LaunchArgs& la, void*, uint64_t, void* stream) { return gr_run<kDx>(la, (cudaStream_t)stream); }
mtl_status gemm_grouped_dw_run(const LaunchArgs& la, void*, uint64_t, void* stream) { return gr_run<kDw>(la, (cudaStream_t)stream); }

}  // namespace mtl
