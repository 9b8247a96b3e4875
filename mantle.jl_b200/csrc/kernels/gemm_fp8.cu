// Matrix products of 8-bit floating point with one scale per block of 128 values
// along K, on the 5th-generation tensor cores:
//
//   C[m, n] = sum_kb sA[kb, m] * sB[kb, n] * ( sum_{k in block kb} A[m, k] * B[n, k] )
//
// A: M rows of K codes, B: N rows of K codes (both e4m3 or e5m2, rows K rounded up
// to 16 bytes apart, as quantize_fp8 writes them), sA: (K blocks, M), sB: one scale
// per 128 x 128 block (N blocks, K blocks) or per row (K blocks, N); C fp32 or bf16.
// The same kernels run a batch of products and products grouped by expert
// (gemm_grouped_fp8: rows offsets[e] .. offsets[e + 1] of A times B[e]). Two forms for
// few rows follow the tiles below.
//
// The scales are arbitrary fp32 values, so a block's products cannot simply
// accumulate in tensor memory: each K block of 128 is one chain of four
// tcgen05.mma (kind::f8f6f4, K = 32) into its own accumulator, and eight warps
// read it back (tcgen05.ld), multiply by the scales and add to fp32 sums in
// registers, rounding to nearest, while the tensor core runs the next K block
// into another accumulator. A K block of a 128 x 256 tile is 512 cycles of MMAs, but
// with its loads and the hand-offs of the two accumulators that fit it takes about 860
// with nothing to add, and with the sums about 1050: 8192 cubed takes 536 us in a burst
// (2050 TFLOP/s) and 622 to 635 in a long run, which the power cap holds to that.
//
// One persistent CTA per SM, three warpgroups; the first gives registers up
// (setmaxnreg) so that the sums of the other two stay in theirs:
//   warp 0      TMA producer: per K block 128 rows of A and BN rows of B, 128 bytes
//               each (128-byte swizzle), into a ring of stages;
//   warp 1      owns the tensor memory, one thread issues the MMAs;
//   warp 2      brings the scales of each K block to shared memory (cp.async), ahead;
//   warps 4-11  the scaled sums: warp w reads lanes 32 (w % 4) .., half of BN columns.
// Rows of a partial tile are loaded in boxes of 32, so that a group of a few rows
// reads few; what the skipped rows hold only reaches rows that are not stored.
//
// A dense product of fewer tiles than SMs is split along K over a cluster of CTAs, one
// tile a cluster: each leaves its sums in its shared memory, and the cluster's warps
// add them in rank order (distributed shared memory) and store them.
//
// Waits are bounded; one that runs out makes the CTA wind down, wait for its own
// loads and MMAs in flight, free its tensor memory and return.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../mtl_internal.hpp"
#include "tc_groups.cuh"

namespace mtl {

constexpr int kF8Threads = 384, kF8M = 128, kF8K = 128;
// Registers a thread of the first / the other warpgroups. The kernels are compiled for the
// 168 that both start with: those of 256 columns spill 8 to 60 bytes a thread.
constexpr int kF8FewRegs = 56, kF8ManyRegs = 224;
constexpr int kF8GroupM = 16;  // row tiles per raster group of a dense product

// A stage less than there would be room for, so that rows leave in pieces of 128 bytes
// (store_rows): the warps that store are the ones that sum, and every tile waits for them.
// 4096 x 4096, us, this way, with the pieces of 64 bytes that leave room for the fourth
// stage, and with those and three stages: K = 512 in fp32 27.6, 30.4 and 30.4, in bf16 21.8, 24.5
// and 23.7; K = 2048 with row scales 69.4, 76.2 and 73.2; K = 4096 79.3, 81.6 and 80.3. With two
// stages K = 4096 takes 92.
template <int BN>
struct F8Cfg {
  static constexpr int kStages = BN == 256 ? 3 : BN == 128 ? 5 : 7;
  static constexpr int kAcc = BN == 256 ? 2 : 4;  // accumulators of BN columns
  static constexpr uint32_t kTmemCols = kAcc * BN;
  static constexpr uint32_t kAStage = kF8M * kF8K, kStageBytes = kAStage + BN * kF8K;
};
constexpr int kF8Scales = 2;  // groups of four K blocks whose scales are on their way or in use
struct F8None {};
template <bool GROUPED, bool ROWB>
struct F8Shared {
  uint4 stage[8][2 * kStageWords];  // per warp of sums: output rows on their way out
  alignas(16) float sa[kF8Scales][4][kF8M];            // K blocks' scales of the tile's rows of A
  alignas(16) float sb[kF8Scales][4][ROWB ? 256 : 4];  // and of its rows of B, or of its 128-row blocks
  uint64_t full[8], empty[8], tfull[4], tempty[4], sfull[kF8Scales], sempty[kF8Scales], drain;
  uint32_t tmem;
  int abort;
  typename std::conditional<GROUPED, GroupTable, F8None>::type groups;
};
template <int BN, bool GROUPED, bool ROWB>
constexpr int f8_smem() {
  return F8Cfg<BN>::kStages * (int)F8Cfg<BN>::kStageBytes + (int)sizeof(F8Shared<GROUPED, ROWB>) + 1024;
}

struct F8Args {
  void* C;
  const float *sA, *sB;
  const int* offsets;  // grouped: groups + 1 row offsets
  int M, N, K;         // M: rows of A in all (grouped) or per product
  int batch;           // products or groups
  int kblocks, nblocks;
  uint32_t idesc;
  int a_box;  // rows per TMA box of A
  int vec;    // rows of C start on 16 bytes
  int splits;  // CTAs a tile (a cluster), SPLIT kernels
  int stall;   // the CTA whose producer stops after one K block, see take_stall
};

__device__ int g_fp8_timeouts;

__device__ __forceinline__ void tc_mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Four bytes to shared memory without a register; they land before the barrier's
// phase completes (cp_async_arrive, one arrival per lane).
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// a += p * s, volatile so that it stays between the loads from tensor memory that it
// is placed between. (The packed form, fma.rn.f32x2, was 4 % slower at 8192 cubed.)
__device__ __forceinline__ void scaled_add(float& a, uint32_t p, float s) {
  asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(a) : "f"(__uint_as_float(p)), "f"(s));
}
// (x, y) times s as one packed operation.
__device__ __forceinline__ void scale2(float& x, float& y, float s) {
  asm("{ .reg .b64 a, b; mov.b64 a, {%0, %1}; mov.b64 b, {%2, %2}; mul.rn.f32x2 a, a, b; mov.b64 {%0, %1}, a; }"
      : "+f"(x), "+f"(y)
      : "f"(s));
}
__device__ __forceinline__ void tmem_ld_nowait(uint32_t addr, uint32_t (&r)[32]) { tmem_ld32_nowait(addr, r); }
__device__ __forceinline__ void tmem_ld_nowait(uint32_t addr, uint32_t (&r)[16]) { tmem_ld16_nowait(addr, r); }
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// A tile's place: rows row0 .. of operand A in slice a_b, columns n0 .. of operand
// B in slice b_b, C's first row, the first element of A's scales, valid rows.
struct F8Tile {
  int a_row, a_b, b_b, n0, rows;
  int64_t crow, sa;
};

template <bool GROUPED>
struct F8Walk {
  GroupWalk g;
  template <typename G>  // the group table, grouped
  __device__ __forceinline__ F8Tile find(const F8Args& p, const G* groups, int64_t t, int tiles_m, int tiles_n, int bn) {
    F8Tile c;
    if constexpr (GROUPED) {
      g.find(groups, (int)t, tiles_n, kF8M, bn, &c.a_row, &c.rows, &c.n0);
      c.a_b = 0;
      c.b_b = g.e;
      c.crow = c.sa = c.a_row;
    } else {
      const int64_t per = (int64_t)tiles_m * tiles_n;
      c.a_b = c.b_b = (int)(t / per);
      const int r = (int)(t % per), group = r / (kF8GroupM * tiles_n), first = group * kF8GroupM;
      const int size = min(kF8GroupM, tiles_m - first), in = r - group * kF8GroupM * tiles_n;
      c.a_row = (first + in % size) * kF8M;
      c.n0 = in / size * bn;
      c.rows = p.M - c.a_row;
      c.crow = (int64_t)c.a_b * p.M + c.a_row;
      c.sa = (int64_t)c.a_b * p.kblocks * p.M + c.a_row;
    }
    c.rows = min(c.rows, kF8M);
    return c;
  }
};

__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %4, %5; ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a]; }"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr), "r"(rank));
  return v;
}
// BN columns a tile; GROUPED: rows by offsets; ROWB: B's scales per row (else
// 128 x 128); SPLIT: a cluster a tile, the K blocks split over its CTAs; OUT: float
// or bf16.
template <int BN, bool GROUPED, bool ROWB, bool SPLIT, typename OUT>
__global__ void __launch_bounds__(kF8Threads, 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const F8Args p) {
  using Cfg = F8Cfg<BN>;
  constexpr int kStages = Cfg::kStages, kAcc = Cfg::kAcc, kCols = BN / 2;
  extern __shared__ unsigned char f8_raw[];
  unsigned char* ring =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(f8_raw) + 1023) & ~uintptr_t(1023));
  auto* sh = reinterpret_cast<F8Shared<GROUPED, ROWB>*>(ring + kStages * Cfg::kStageBytes);
  volatile int* abort = &sh->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(smem_u32(&sh->tfull[a]), 1);
      mbar_init(smem_u32(&sh->tempty[a]), 8);
    }
    for (int a = 0; a < kF8Scales; ++a) {
      mbar_init(smem_u32(&sh->sfull[a]), 32);
      mbar_init(smem_u32(&sh->sempty[a]), 8);
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
  if constexpr (GROUPED) build_groups(&sh->groups, p.offsets, p.batch, p.M, kF8M);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;

  const int tiles_m = (p.M + kF8M - 1) / kF8M, tiles_n = (p.N + BN - 1) / BN;
  int64_t ntiles = (int64_t)tiles_m * tiles_n * p.batch;
  if constexpr (GROUPED) ntiles = (int64_t)sh->groups.cum[p.batch] * tiles_n;
  F8Walk<GROUPED> walk;
  // this CTA's tiles and K blocks
  const int rank = SPLIT ? (int)blockIdx.x % p.splits : 0;
  const int64_t t0 = SPLIT ? blockIdx.x / p.splits : blockIdx.x, tstep = SPLIT ? ntiles : gridDim.x;
  const int kbeg = SPLIT ? (int)((int64_t)p.kblocks * rank / p.splits) : 0;
  const int kend = SPLIT ? (int)((int64_t)p.kblocks * (rank + 1) / p.splits) : p.kblocks;

  // 384 threads start with 168 registers each: 128 x 56 + 256 x 224 = 384 x 168
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8FewRegs));
    if (warp == 0) {
      // ── TMA producer (the whole warp waits, one lane issues) ──
      int s = 0;
      uint32_t ph = 0;
      int64_t issued = 0;
      bool ok = true;
      const bool stalls = (int)blockIdx.x == p.stall;
      for (int64_t t = t0; ok && t < ntiles; t += tstep) {
        const F8Tile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n, BN);
        const int boxes = (c.rows + p.a_box - 1) / p.a_box;
        const uint32_t bytes = (uint32_t)(boxes * p.a_box * kF8K + BN * kF8K);
        const int last = stalls ? min(kend, kbeg + 1) : kend;
        for (int kb = kbeg; kb < last; ++kb) {
          ok = wait_warp(smem_u32(&sh->empty[s]), ph ^ 1, abort, &g_fp8_timeouts);
          if (!ok) break;
          if (elect_one()) {
            const uint32_t fb = smem_u32(&sh->full[s]), dst = smem_u32(ring) + (uint32_t)(s * Cfg::kStageBytes);
            mbar_expect_tx(fb, bytes);
            tma_load_3d(dst + Cfg::kAStage, &tmB, kb * kF8K, c.n0, c.b_b, fb);
            for (int r = 0; r < boxes; ++r)
              tma_load_3d(dst + r * p.a_box * kF8K, &tmA, kb * kF8K, c.a_row + r * p.a_box, c.a_b, fb);
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
      // ── MMA issuer (the whole warp waits, one lane issues) ──
      int s = 0, a = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      // both operands K-major: rows of 128 bytes, 8-row groups 1024 bytes apart; a K = 32
      // slice is 32 bytes further along the swizzled row
      const uint64_t a0 = smem_desc(smem_u32(ring), 16, 1024), b0 = smem_desc(smem_u32(ring) + Cfg::kAStage, 16, 1024);
      for (int64_t t = t0; ok && t < ntiles; t += tstep) {
        for (int kb = kbeg; kb < kend; ++kb) {
          // the loads were there long before; the accumulator is what the MMAs wait for
          ok = wait_warp(smem_u32(&sh->full[s]), ph, abort, &g_fp8_timeouts) &&
               wait_warp(smem_u32(&sh->tempty[a]), aph ^ 1, abort, &g_fp8_timeouts);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t d = tmem + (uint32_t)(a * BN);
            const uint64_t ad = a0 + (uint64_t)(s * (Cfg::kStageBytes >> 4)), bd = b0 + (uint64_t)(s * (Cfg::kStageBytes >> 4));
#pragma unroll
            for (int kk = 0; kk < kF8K / 32; ++kk) tc_mma_f8(d, ad + kk * 2, bd + kk * 2, p.idesc, kk != 0);
            tc_commit(smem_u32(&sh->empty[s]));
            tc_commit(smem_u32(&sh->tfull[a]));
          }
          __syncwarp();
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
          if (++a == kAcc) {
            a = 0;
            aph ^= 1;
          }
        }
      }
      if (!ok) drain_mmas<false>(smem_u32(&sh->drain));
    } else if (warp == 2) {
      // ── scales: a K block's 128 + BN (or its 128-row blocks') into a ring of their own ──
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int64_t t = t0; ok && t < ntiles; t += tstep) {
        const F8Tile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n, BN);
        const float* sa = p.sA + c.sa;
        const float* sb = ROWB ? p.sB + (int64_t)c.b_b * p.kblocks * p.N + c.n0
                               : p.sB + ((int64_t)c.b_b * p.nblocks + c.n0 / 128) * p.kblocks;
        const int cols = min(BN, p.N - c.n0);
        for (int kb0 = kbeg; kb0 < kend; kb0 += 4) {
          ok = wait_warp(smem_u32(&sh->sempty[s]), ph ^ 1, abort, &g_fp8_timeouts);
          if (!ok) break;
          for (int j = 0; j < min(4, kend - kb0); ++j) {
            const uint32_t da = smem_u32(sh->sa[s][j]), db = smem_u32(sh->sb[s][j]);
            const int64_t kb = kb0 + j;
#pragma unroll
            for (int i = 0; i < kF8M / 32; ++i)
              if (i * 32 + lane < c.rows) cp_async4(da + (i * 32 + lane) * 4, sa + kb * p.M + i * 32 + lane);
            if (ROWB) {
#pragma unroll
              for (int i = 0; i < BN / 32; ++i)
                if (i * 32 + lane < cols) cp_async4(db + (i * 32 + lane) * 4, sb + kb * p.N + i * 32 + lane);
            } else if (lane * 128 < cols) {
              cp_async4(db + lane * 4, sb + (int64_t)lane * p.kblocks + kb);
            }
          }
          cp_async_arrive(smem_u32(&sh->sfull[s]));
          if (++s == kF8Scales) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if constexpr (SPLIT) {  // the two meetings of the cluster, see the other warps
      cluster_sync();
      cluster_sync();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8ManyRegs));
    // ── scaled sums: warp reads TMEM lanes 32 q .. +32, columns half * kCols .. ──
    const int q = warp & 3, half = (warp - 4) / 4;
    int a = 0, s = 0;
    uint32_t aph = 0, sph = 0;
    bool ok = true;
    for (int64_t t = t0; ok && t < ntiles; t += tstep) {
      const F8Tile c = walk.find(p, &sh->groups, t, tiles_m, tiles_n, BN);
      const int row = q * 32 + lane, col = c.n0 + half * kCols;
      const bool busy = q * 32 < c.rows;  // uniform in the warp
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
      // K block kb's accumulator is there, and every fourth time the next four blocks' scales
      auto arrived = [&](int kb) {
        bool here = ((kb - kbeg) & 3) != 0 || wait_warp(smem_u32(&sh->sfull[s]), sph, abort, &g_fp8_timeouts);
        here = here && wait_warp(smem_u32(&sh->tfull[a]), aph, abort, &g_fp8_timeouts);
        tc_fence_after();
        return here;
      };
      auto give_back = [&](uint64_t* bar) {  // after every lane's last use
        __syncwarp();
        if (elect_one()) mbar_arrive(smem_u32(bar));
      };
      auto next_acc = [&]() {
        if (++a == kAcc) {
          a = 0;
          aph ^= 1;
        }
      };
      auto next_scales = [&](int kb) {  // after K block kb
        if (((kb - kbeg) & 3) == 3 || kb + 1 == kend) {
          give_back(&sh->sempty[s]);
          if (++s == kF8Scales) {
            s = 0;
            sph ^= 1;
          }
        }
      };
      if (!busy) {
        for (int kb = kbeg; ok && kb < kend; ++kb) {
          ok = arrived(kb);
          if (!ok) break;
          give_back(&sh->tempty[a]);
          next_acc();
          next_scales(kb);
        }
        continue;
      }
      // Chunks of kW columns, two in registers: while one is multiplied and added the
      // next one is on its way from tensor memory.
      constexpr int kW = kCols / 2 < 32 ? kCols / 2 : 32, kChunks = kCols / kW;
      uint32_t r[2][kW];
      const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * kCols);
#pragma unroll 1
      for (int kb = kbeg; kb < kend; ++kb) {
        ok = arrived(kb);
        if (!ok) break;
        const uint32_t from = lanes + (uint32_t)(a * BN);
        tmem_ld_nowait(from, r[0]);
        const float sr = ROWB ? sh->sa[s][(kb - kbeg) & 3][row] : sh->sa[s][(kb - kbeg) & 3][row] * sh->sb[s][(kb - kbeg) & 3][BN == 256 ? half : 0];
        const float* sb = sh->sb[s][(kb - kbeg) & 3] + half * kCols;
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
          tmem_wait_ld(r[ch & 1]);
          if (ch + 1 < kChunks) {
            tmem_ld_nowait(from + (uint32_t)((ch + 1) * kW), r[(ch + 1) & 1]);
          } else {
            tc_fence_before();
            give_back(&sh->tempty[a]);
            next_acc();
          }
#pragma unroll
          for (int i = 0; i < kW; i += 4) {
            float4 f = make_float4(sr, sr, sr, sr);
            if (ROWB) {  // the same word in every lane; two products an instruction
              const float4 b = *reinterpret_cast<const float4*>(sb + ch * kW + i);
              f = b;
              scale2(f.x, f.y, sr);
              scale2(f.z, f.w, sr);
            }
            scaled_add(acc[ch * kW + i], r[ch & 1][i], f.x);
            scaled_add(acc[ch * kW + i + 1], r[ch & 1][i + 1], f.y);
            scaled_add(acc[ch * kW + i + 2], r[ch & 1][i + 2], f.z);
            scaled_add(acc[ch * kW + i + 3], r[ch & 1][i + 3], f.w);
          }
        }
        next_scales(kb);
      }
      if constexpr (SPLIT) {  // the ring is free: every load landed and every MMA is done
        // four columns of a row a word, the rows of a word's columns next to one another
        float4* part = reinterpret_cast<float4*>(ring) + (half * kCols / 4) * kF8M + row;
        if (ok) {
#pragma unroll
          for (int i = 0; i < kCols; i += 4) part[i / 4 * kF8M] = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        } else {  // a CTA that gave up: the tile is NaN, not part of a sum
          const float lost = __int_as_float(0x7fc00000);
#pragma unroll 1
          for (int i = 0; i < kCols; i += 4) part[i / 4 * kF8M] = make_float4(lost, lost, lost, lost);
        }
        break;
      }
      if (!ok) break;
      constexpr int kOut = kCols * sizeof(OUT) < 128 ? kCols : 128 / sizeof(OUT);  // columns a piece
      OUT* out = static_cast<OUT*>(p.C) + (c.crow + q * 32) * p.N;
#pragma unroll
      for (int i = 0; i < kCols; i += kOut)
        if (col + i < p.N)
          store_rows(sh->stage[warp - 4], lane, c.rows - q * 32, out, p.N, col + i, p.vec,
                     reinterpret_cast<const float(&)[kOut]>(acc[i]));
    }
    if constexpr (SPLIT) {
      cluster_sync();  // every CTA of the tile has its sums in shared memory, column by column
      const F8Tile c = walk.find(p, &sh->groups, t0, tiles_m, tiles_n, BN);
      constexpr int kOut = 64 / sizeof(OUT);
      const int quarters = (c.rows + 31) / 32, pieces = (min(BN, p.N - c.n0) + kOut - 1) / kOut;
      for (int i = rank * 8 + warp - 4; i < quarters * pieces; i += p.splits * 8) {
        const int rq = i % quarters, col = i / quarters * kOut;
        const uint32_t at = smem_u32(ring) + (uint32_t)((col / 4 * kF8M + rq * 32 + lane) * 16);
        float v[kOut];
#pragma unroll
        for (int k = 0; k < kOut; ++k) v[k] = 0.0f;
        for (int r = 0; r < p.splits; ++r) {
          float4 u[kOut / 4];
#pragma unroll
          for (int k = 0; k < kOut / 4; ++k) u[k] = ld_cluster(at + (uint32_t)(k * kF8M * 16), (uint32_t)r);
#pragma unroll
          for (int k = 0; k < kOut / 4; ++k) {
            v[4 * k] += u[k].x;
            v[4 * k + 1] += u[k].y;
            v[4 * k + 2] += u[k].z;
            v[4 * k + 3] += u[k].w;
          }
        }
        store_rows(sh->stage[warp - 4], lane, c.rows - rq * 32, static_cast<OUT*>(p.C) + (c.crow + rq * 32) * p.N, p.N,
                   c.n0 + col, p.vec, v);
      }
      cluster_sync();  // no CTA leaves while others read its sums
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kTmemCols) : "memory");
}

// ── groups of a few rows of A ───────────────────────────────────────────────
// As the tiles above, with the roles of the operands changed: 256 rows of B (two runs of
// 128) are the MMA's M operand and NT rows of a group its N operand, so a K block takes a
// quarter of the MMAs or less, and its sums, transposed in tensor memory (a lane has one
// column of C), are NT multiplications and additions a lane instead of 128 of which few
// are stored. Eight K blocks' sums fit in tensor memory, so they and their scales are
// handed over four at a time, in one wait each (128 rows over 64 experts of 4096 x 2048:
// 85.8 -> 85.1 us against a wait for every block; 1024 rows, 2048 x 2048: 49.6 -> 49.0).
constexpr int kSlim = 32;  // rows of a group a tile
template <int NT>
struct SlimF8 {
  static constexpr uint32_t kBStage = 256 * kF8K, kXStage = NT * kF8K, kStageBytes = kBStage + kXStage;
  static constexpr int kStages = 196608 / (int)kStageBytes;
  static constexpr uint32_t kTmemCols = 2 * 4 * 2 * NT;  // two groups of four K blocks of two runs
};
template <int NT>
struct SlimF8Shared {
  alignas(16) float sa[2][4][NT];  // two groups of four K blocks: the rows' scales
  alignas(16) float sb[2][4][4];   // and the two runs'
  uint64_t full[8], empty[8], tfull[2], tempty[2], sfull[2], sempty[2], drain;
  uint32_t tmem;
  int abort;
  GroupTable groups;
};
template <int NT>
constexpr int slim_f8_smem() {
  return SlimF8<NT>::kStages * (int)SlimF8<NT>::kStageBytes + (int)sizeof(SlimF8Shared<NT>) + 1024;
}

template <int NT, typename OUT>
__global__ void __launch_bounds__(kF8Threads, 1)
    gemm_fp8_slim_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const F8Args p) {
  using Cfg = SlimF8<NT>;
  constexpr int kStages = Cfg::kStages, BN = 256;
  extern __shared__ unsigned char f8_raw[];
  unsigned char* ring =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(f8_raw) + 1023) & ~uintptr_t(1023));
  auto* sh = reinterpret_cast<SlimF8Shared<NT>*>(ring + kStages * Cfg::kStageBytes);
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
      mbar_init(smem_u32(&sh->sfull[a]), 32);
      mbar_init(smem_u32(&sh->sempty[a]), 8);
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
  build_groups(&sh->groups, p.offsets, p.batch, p.M, NT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  const int tiles_n = (p.N + BN - 1) / BN, ntiles = sh->groups.cum[p.batch] * tiles_n;
  GroupWalk walk;
  int row0, rows, n0;

  if (warp == 0) {
    // ── TMA producer ──
    int s = 0;
    uint32_t ph = 0;
    int64_t issued = 0;
    bool ok = true;
    const bool stalls = (int)blockIdx.x == p.stall;
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      walk.find(&sh->groups, t, tiles_n, NT, BN, &row0, &rows, &n0);
      const int last = stalls ? min(p.kblocks, 1) : p.kblocks;
      for (int kb = 0; kb < last; ++kb) {
        ok = wait_warp(smem_u32(&sh->empty[s]), ph ^ 1, abort, &g_fp8_timeouts);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t fb = smem_u32(&sh->full[s]), dst = smem_u32(ring) + (uint32_t)(s * Cfg::kStageBytes);
          mbar_expect_tx(fb, Cfg::kStageBytes);
          tma_load_3d(dst, &tmB, kb * kF8K, n0, walk.e, fb);
          // rows behind the group's feed sums that are not stored
          tma_load_3d(dst + Cfg::kBStage, &tmA, kb * kF8K, row0, 0, fb);
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
    int s = 0, a = 0;
    uint32_t ph = 0, aph = 0;
    bool ok = true;
    const uint64_t b0 = smem_desc(smem_u32(ring), 16, 1024), x0 = smem_desc(smem_u32(ring) + Cfg::kBStage, 16, 1024);
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      for (int kb = 0; kb < p.kblocks; ++kb) {
        ok = wait_warp(smem_u32(&sh->full[s]), ph, abort, &g_fp8_timeouts) &&
             ((kb & 3) != 0 || wait_warp(smem_u32(&sh->tempty[a]), aph ^ 1, abort, &g_fp8_timeouts));
        if (!ok) break;
        tc_fence_after();
        const bool last = (kb & 3) == 3 || kb + 1 == p.kblocks;  // of its group
        if (elect_one()) {
          const uint32_t d = tmem + (uint32_t)((a * 4 + (kb & 3)) * 2 * NT);
          const uint64_t off = (uint64_t)(s * (Cfg::kStageBytes >> 4));
#pragma unroll
          for (int kk = 0; kk < kF8K / 32; ++kk)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              tc_mma_f8(d + (uint32_t)(r * NT), b0 + off + r * (Cfg::kBStage / 2 >> 4) + kk * 2, x0 + off + kk * 2, p.idesc, kk != 0);
          tc_commit(smem_u32(&sh->empty[s]));
          if (last) tc_commit(smem_u32(&sh->tfull[a]));
        }
        __syncwarp();
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
        if (last && ++a == 2) {
          a = 0;
          aph ^= 1;
        }
      }
    }
    if (!ok) drain_mmas<false>(smem_u32(&sh->drain));
  } else if (warp == 2) {
    // ── scales, four K blocks at a time ──
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      walk.find(&sh->groups, t, tiles_n, NT, BN, &row0, &rows, &n0);
      const float* sb = p.sB + ((int64_t)walk.e * p.nblocks + n0 / 128) * p.kblocks;
      for (int kb0 = 0; kb0 < p.kblocks; kb0 += 4) {
        ok = wait_warp(smem_u32(&sh->sempty[s]), ph ^ 1, abort, &g_fp8_timeouts);
        if (!ok) break;
        for (int j = 0; j < min(4, p.kblocks - kb0); ++j) {
          const int64_t kb = kb0 + j;
#pragma unroll
          for (int i = 0; i < NT / 32; ++i)
            if (i * 32 + lane < rows) cp_async4(smem_u32(&sh->sa[s][j][i * 32 + lane]), p.sA + kb * p.M + row0 + i * 32 + lane);
          if (lane < 2 && n0 + lane * 128 < p.N) cp_async4(smem_u32(&sh->sb[s][j][lane]), sb + (int64_t)lane * p.kblocks + kb);
        }
        cp_async_arrive(smem_u32(&sh->sfull[s]));
        if (++s == 2) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= 4) {
    // ── scaled sums: a warp has 32 columns of C, run (warp - 4) / 4 ──
    const int q = warp & 3, run = (warp - 4) / 4;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(run * NT);
    int a = 0;  // the group in hand, of scales and of sums alike
    uint32_t ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
      walk.find(&sh->groups, t, tiles_n, NT, BN, &row0, &rows, &n0);
      const int col = n0 + run * 128 + q * 32 + lane;
      float acc[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i] = 0.0f;
      for (int kb = 0; kb < p.kblocks; kb += 4) {
        ok = wait_warp(smem_u32(&sh->sfull[a]), ph, abort, &g_fp8_timeouts) &&
             wait_warp(smem_u32(&sh->tfull[a]), ph, abort, &g_fp8_timeouts);
        if (!ok) break;
        tc_fence_after();
        const int blocks = min(4, p.kblocks - kb);
#pragma unroll
        for (int c = 0; c < NT; c += 16) {
          if (c >= rows) break;  // uniform in the CTA
          uint32_t r[4][16];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < blocks) tmem_ld16_nowait(lanes + (uint32_t)((a * 4 + j) * 2 * NT + c), r[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= blocks) break;
            const float sb = sh->sb[a][j][run];
            const float4* sa = reinterpret_cast<const float4*>(&sh->sa[a][j][c]);
            float4 f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = sa[i];
            tmem_wait_ld(r[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              acc[c + 4 * i] = fmaf(__uint_as_float(r[j][4 * i]), f[i].x * sb, acc[c + 4 * i]);
              acc[c + 4 * i + 1] = fmaf(__uint_as_float(r[j][4 * i + 1]), f[i].y * sb, acc[c + 4 * i + 1]);
              acc[c + 4 * i + 2] = fmaf(__uint_as_float(r[j][4 * i + 2]), f[i].z * sb, acc[c + 4 * i + 2]);
              acc[c + 4 * i + 3] = fmaf(__uint_as_float(r[j][4 * i + 3]), f[i].w * sb, acc[c + 4 * i + 3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (elect_one()) {
          mbar_arrive(smem_u32(&sh->tempty[a]));
          mbar_arrive(smem_u32(&sh->sempty[a]));
        }
        if (++a == 2) {
          a = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
      if (col < p.N) {
        OUT* out = static_cast<OUT*>(p.C) + (int64_t)row0 * p.N + col;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < rows) {
            if constexpr (sizeof(OUT) == 4)
              out[(int64_t)i * p.N] = acc[i];
            else
              out[(int64_t)i * p.N] = __float2bfloat16_rn(acc[i]);
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

// ── few rows of A: a decode step ────────────────────────────────────────────
// With M <= 16 the product is a read of B. mma.sync takes its operands from
// registers, so the codes go from global memory straight into them: a warp holds 16
// rows of B as the MMA's A operand and the rows of A as its 8 columns. The K index is
// permuted alike on both sides (a lane's 16-byte word feeds four K = 32 slices' worth
// of fragments of its row), so every load is a 16-byte word and no shuffle or shared
// memory is needed. The CTA's eight warps take the K blocks in turn, kAhead at a time
// to keep loads in flight, and their sums meet in shared memory in warp order.
// Blocks that end by K are loaded without a branch (a test in each load kept them from
// being in flight together: 65536 x 4096 at one row 63 us, 49 without = 5.5 TB/s).
// At one row, 8192 x 4096: 8.2 us, 14.6 with the tiles above.
constexpr int kFewThreads = 256, kFewRows = 16;

template <bool A5, bool B5>  // A: the MMA's first operand (B's codes), e5m2 or e4m3
__device__ __forceinline__ void mma_f8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
#define MTL_MMA_F8(ta, tb)                                                                                       \
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32." ta "." tb ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " \
               "{%0,%1,%2,%3};"                                                                                  \
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                  \
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if constexpr (A5 && B5)
    MTL_MMA_F8("e5m2", "e5m2");
  else if constexpr (A5)
    MTL_MMA_F8("e5m2", "e4m3");
  else if constexpr (B5)
    MTL_MMA_F8("e4m3", "e5m2");
  else
    MTL_MMA_F8("e4m3", "e4m3");
#undef MTL_MMA_F8
}

// Sixteen codes of a row from column k on; those at or past K are zeros, whatever the
// row's padding holds.
__device__ __forceinline__ uint4 codes16(const uint8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i / 4] |= (uint32_t)row[k + i] << (i % 4 * 8);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int MT, bool ROWB, bool A5, bool B5, typename OUT>  // MT: groups of eight rows of A
__global__ void __launch_bounds__(kFewThreads, 2)
    gemm_fp8_few_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ B, const F8Args p) {
  constexpr int kAhead = 2, kWarps = kFewThreads / 32;
  __shared__ float sums[kWarps][MT][16][8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int ntiles = (p.N + 15) / 16, b = blockIdx.x / ntiles, n0 = blockIdx.x % ntiles * 16;
  const int64_t ld = (p.K + 15) / 16 * 16;
  const uint8_t* rows_b[2];  // past N: the last row, its sums are not stored
#pragma unroll
  for (int h = 0; h < 2; ++h) rows_b[h] = B + ((int64_t)b * p.N + min(n0 + g + h * 8, p.N - 1)) * ld;
  const float* sa = p.sA + (int64_t)b * p.kblocks * p.M;
  const float* sb = ROWB ? p.sB + (int64_t)b * p.kblocks * p.N : p.sB + ((int64_t)b * p.nblocks + n0 / 128) * p.kblocks;
  float acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[m][i] = 0.0f;

  const uint8_t* rows_a[MT];  // past M: the last row, its sums are not stored
  int cols_a[MT][2];          // the rows of A this lane's sums belong to
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    rows_a[m] = A + ((int64_t)b * p.M + min(m * 8 + g, p.M - 1)) * ld;
#pragma unroll
    for (int c = 0; c < 2; ++c) cols_a[m][c] = min(m * 8 + t * 2 + c, p.M - 1);
  }
  const int rows_sb[2] = {min(n0 + g, p.N - 1), min(n0 + g + 8, p.N - 1)};

  // U K blocks from kb on, kWarps apart; WHOLE: every one of them ends by K
  auto blocks = [&](int kb, auto u_c, auto whole_c) {
    constexpr int U = decltype(u_c)::value;
    constexpr bool WHOLE = decltype(whole_c)::value;
    uint4 wb[U][2][2], wa[U][MT][2];
    float fa[U][MT][2], fb[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = kb + u * kWarps, k = at * 128 + t * 16;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          wb[u][h][e] = WHOLE ? __ldg(reinterpret_cast<const uint4*>(rows_b[h] + k + e * 64)) : codes16(rows_b[h], k + e * 64, p.K);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          wa[u][m][e] = WHOLE ? __ldg(reinterpret_cast<const uint4*>(rows_a[m] + k + e * 64)) : codes16(rows_a[m], k + e * 64, p.K);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) fa[u][m][c] = __ldg(sa + (int64_t)at * p.M + cols_a[m][c]);
#pragma unroll
      for (int h = 0; h < 2; ++h) fb[u][h] = __ldg(ROWB ? sb + (int64_t)at * p.N + rows_sb[h] : sb + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float d[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint4 x = wb[u][0][e], y = wb[u][1][e], z = wa[u][m][e];
          mma_f8<B5, A5>(d, x.x, y.x, x.y, y.y, z.x, z.y);
          mma_f8<B5, A5>(d, x.z, y.z, x.w, y.w, z.z, z.w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(d[i], fa[u][m][i & 1] * fb[u][i / 2], acc[m][i]);
      }
  };
  const int whole = p.K / 128;
  int kb = warp;
  for (; kb + (kAhead - 1) * kWarps < whole; kb += kWarps * kAhead)
    blocks(kb, std::integral_constant<int, kAhead>(), std::true_type());
  for (; kb < whole; kb += kWarps) blocks(kb, std::integral_constant<int, 1>(), std::true_type());
  if (kb < p.kblocks) blocks(kb, std::integral_constant<int, 1>(), std::false_type());  // the last one, short
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[warp][m][g + i / 2 * 8][t * 2 + (i & 1)] = acc[m][i];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 128; o += kFewThreads) {
    const int n = o % 16, m = o / 16;  // sixteen neighbouring columns of a row of C
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sums[w][m / 8][n][m % 8];
    if (m < p.M && n0 + n < p.N) {
      OUT* c = static_cast<OUT*>(p.C) + ((int64_t)b * p.M + m) * p.N + n0 + n;
      if constexpr (sizeof(OUT) == 4)
        *c = v;
      else
        *c = __float2bfloat16_rn(v);
    }
  }
}

// ── host side ───────────────────────────────────────────────────────────────
static int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Codes as bytes: {K, rows, slices}, rows K rounded up to 16 bytes apart, a box of
// 128 bytes x box_rows, 128-byte swizzle, zeros outside.
static mtl_status make_code_map(CUtensorMap* map, const void* base, int64_t K, int64_t rows, int64_t slices, int box_rows) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return fail(MTL_ERR_CUDA, "gemm_fp8: cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)slices};
  cuuint64_t strides[2] = {(cuuint64_t)up16(K), (cuuint64_t)(up16(K) * rows)};
  cuuint32_t box[3] = {128, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MTL_ERR_ARGUMENT, "gemm_fp8: tensor map rejected (CUresult %d)", (int)r);
  return MTL_OK;
}

static std::atomic<int> g_fp8_stalls{0};
void fp8_inject_stall(int launches) { g_fp8_stalls.store(launches > 0 ? launches : 0); }
cudaError_t fp8_set_wait_limit(unsigned long long ns) { return set_wait_limit_this_file(ns); }
int fp8_timeouts(bool reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_fp8_timeouts, sizeof v) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (reset && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_fp8_timeouts, &zero, sizeof zero);
  }
  return v;
}

template <int BN, bool GROUPED, bool ROWB, bool SPLIT, typename OUT>
static cudaError_t fp8_launch(const CUtensorMap& ta, const CUtensorMap& tb, const F8Args& p, int64_t tiles, int sms,
                              int device, cudaStream_t s) {
  auto kernel = gemm_fp8_kernel<BN, GROUPED, ROWB, SPLIT, OUT>;
  constexpr int smem = f8_smem<BN, GROUPED, ROWB>();
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(kernel, smem, device, &done);
  if (e != cudaSuccess) return e;
  // the register split draws on what the block starts with: with less it would wait for good
  static int known = 0;  // registers a thread, once the runtime has said
  int regs = __atomic_load_n(&known, __ATOMIC_RELAXED);
  if (!regs) {
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, kernel)) != cudaSuccess) return e;
    __atomic_store_n(&known, regs = at.numRegs, __ATOMIC_RELAXED);
  }
  if (regs * kF8Threads < 128 * kF8FewRegs + 256 * kF8ManyRegs) return cudaErrorLaunchOutOfResources;
  if constexpr (SPLIT) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.splits));
    cfg.blockDim = dim3(kF8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, ta, tb, p);
  } else {
    kernel<<<(int)std::min<int64_t>(tiles, sms), kF8Threads, smem, s>>>(ta, tb, p);
    return cudaGetLastError();
  }
}
template <int BN, bool GROUPED, bool ROWB, typename OUT>
static cudaError_t fp8_launch_split(const CUtensorMap& ta, const CUtensorMap& tb, const F8Args& p, int64_t tiles, int sms,
                                    int device, cudaStream_t s) {
  if constexpr (!GROUPED)
    if (p.splits > 1) return fp8_launch<BN, GROUPED, ROWB, true, OUT>(ta, tb, p, tiles, sms, device, s);
  return fp8_launch<BN, GROUPED, ROWB, false, OUT>(ta, tb, p, tiles, sms, device, s);
}
template <int BN, bool GROUPED>
static cudaError_t fp8_launch_by(bool rowb, bool bf16, const CUtensorMap& ta, const CUtensorMap& tb, const F8Args& p,
                                 int64_t tiles, int sms, int device, cudaStream_t s) {
  if constexpr (!GROUPED) {
    if (rowb)
      return bf16 ? fp8_launch_split<BN, GROUPED, true, __nv_bfloat16>(ta, tb, p, tiles, sms, device, s)
                  : fp8_launch_split<BN, GROUPED, true, float>(ta, tb, p, tiles, sms, device, s);
  }
  return bf16 ? fp8_launch_split<BN, GROUPED, false, __nv_bfloat16>(ta, tb, p, tiles, sms, device, s)
              : fp8_launch_split<BN, GROUPED, false, float>(ta, tb, p, tiles, sms, device, s);
}

template <int MT, bool ROWB, bool A5, bool B5>
static void fp8_few_by(bool bf16, const uint8_t* A, const uint8_t* B, const F8Args& p, unsigned grid, cudaStream_t s) {
  if (bf16)
    gemm_fp8_few_kernel<MT, ROWB, A5, B5, __nv_bfloat16><<<grid, kFewThreads, 0, s>>>(A, B, p);
  else
    gemm_fp8_few_kernel<MT, ROWB, A5, B5, float><<<grid, kFewThreads, 0, s>>>(A, B, p);
}
template <int MT, bool ROWB>
static cudaError_t fp8_few(bool a5, bool b5, bool bf16, const uint8_t* A, const uint8_t* B, const F8Args& p, cudaStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.batch * ((p.N + 15) / 16));
  if (a5)
    b5 ? fp8_few_by<MT, ROWB, true, true>(bf16, A, B, p, grid, s) : fp8_few_by<MT, ROWB, true, false>(bf16, A, B, p, grid, s);
  else
    b5 ? fp8_few_by<MT, ROWB, false, true>(bf16, A, B, p, grid, s) : fp8_few_by<MT, ROWB, false, false>(bf16, A, B, p, grid, s);
  return cudaGetLastError();
}

template <int NT, typename OUT>
static cudaError_t fp8_launch_slim(const CUtensorMap& ta, const CUtensorMap& tb, const F8Args& p, int64_t tiles, int sms,
                                   int device, cudaStream_t s) {
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(gemm_fp8_slim_kernel<NT, OUT>, slim_f8_smem<NT>(), device, &done);
  if (e != cudaSuccess) return e;
  gemm_fp8_slim_kernel<NT, OUT><<<(int)std::min<int64_t>(tiles, sms), kF8Threads, slim_f8_smem<NT>(), s>>>(ta, tb, p);
  return cudaGetLastError();
}

// What gemm_fp8 and gemm_grouped_fp8 check alike. `rows`: rows of A and C over the
// whole launch; `slices`: products or experts.
static mtl_status fp8_check_common(const char* who, const LaunchArgs& la, const uint64_t* bytes, int64_t batch, int64_t M,
                                   int64_t N, int64_t K, int64_t rows, int bblock, int fa, int fb, int out) {
  if (la.ndim != 1) return fail(MTL_ERR_ARGUMENT, "%s: ndrange must be one-dimensional", who);
  if (M < 0 || N < 0 || K < 0) return fail(MTL_ERR_ARGUMENT, "%s: negative dimension", who);
  if (std::max({M, N, K}) > kMaxSize) return fail(MTL_ERR_UNSUPPORTED, "%s: a dimension above 2^31 - 256", who);
  if (bblock != 1 && bblock != 128)
    return fail(MTL_ERR_ARGUMENT, "%s: B's scales cover 1 or 128 rows each, got %d", who, bblock);
  if ((fa | fb | out) & ~1)
    return fail(MTL_ERR_ARGUMENT, "%s: formats are 0 (e4m3) or 1 (e5m2), the output 0 (fp32) or 1 (bf16), got %d, %d, %d", who, fa, fb, out);
  const int64_t kb = (K + 127) / 128, nb = (N + 127) / 128;
  const uint64_t need[5] = {bytes_of({rows, N, out ? 2 : 4}), bytes_of({rows, up16(K)}), bytes_of({kb, rows, 4}),
                            bytes_of({batch, N, up16(K)}), bytes_of({batch, kb, bblock == 1 ? N : nb, 4})};
  const char* what[5] = {"C", "A", "A's scales", "B", "B's scales"};
  const unsigned align[5] = {out ? 1u : 3u, 15, 3, 15, 3};
  for (int i = 0; i < 5; ++i) {
    if (!la.a[i].ptr && need[i]) return fail(MTL_ERR_ARGUMENT, "%s: %s must be a device buffer", who, what[i]);
    if (bytes[i] && bytes[i] < need[i])
      return fail(MTL_ERR_ARGUMENT, "%s: %s has %llu bytes, the launch touches %llu", who, what[i], (unsigned long long)bytes[i],
                  (unsigned long long)need[i]);
    if (la.a[i].ptr & align[i]) return fail(MTL_ERR_ARGUMENT, "%s: %s must be %u-byte aligned", who, what[i], align[i] + 1);
  }
  if (((M + 31) / 32 + kMaxGroups) * ((N + 63) / 64) > INT_MAX)
    return fail(MTL_ERR_UNSUPPORTED, "%s: more than 2^31 tiles a product", who);
  return MTL_OK;
}

// Arguments: C (B), A (B), sA (B), B (B), sB (B), M, N, K, rows per scale of B, format
// of A, format of B, output type (i); ndrange = batch.
mtl_status gemm_fp8_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int64_t batch = la.nd[0], M = la.a[5].i32;
  if (batch > 65535) return fail(MTL_ERR_UNSUPPORTED, "gemm_fp8: batch above 65535");
  return fp8_check_common("gemm_fp8", la, bytes, batch, M, la.a[6].i32, la.a[7].i32, batch * M, la.a[8].i32, la.a[9].i32,
                          la.a[10].i32, la.a[11].i32);
}

// Arguments: Y (B), X (B), sX (B), W (B), sW (B), offsets (B, i32, groups + 1), T, N, K,
// format of X, format of W, output type (i); ndrange = groups.
mtl_status gemm_grouped_fp8_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int64_t groups = la.nd[0], T = la.a[6].i32;
  if (groups > kMaxGroups) return fail(MTL_ERR_UNSUPPORTED, "gemm_grouped_fp8: more than %d groups", kMaxGroups);
  if (mtl_status st = fp8_check_common("gemm_grouped_fp8", la, bytes, groups, T, la.a[7].i32, la.a[8].i32, T, 128, la.a[9].i32,
                                       la.a[10].i32, la.a[11].i32))
    return st;
  if (la.a[8].i32 == 0) return fail(MTL_ERR_ARGUMENT, "gemm_grouped_fp8: K must be positive");
  if (!la.a[5].ptr || (bytes[5] && bytes[5] < (uint64_t)(groups + 1) * 4) || la.a[5].ptr % 4)
    return fail(MTL_ERR_ARGUMENT, "gemm_grouped_fp8: the offsets are %lld 4-byte aligned Int32 values", (long long)groups + 1);
  return MTL_OK;
}

// Tile width and K parts of a launch, by a model of what was measured: the rounds of
// K blocks, a block's time (a chain of hand-offs between loads, MMAs and sums) 550,
// 420 and 350 ns for 256, 128 and 64 columns; a split costs 3 us and a quarter of a
// microsecond per 32 x 64 sums it adds. It is right to some percent where it was
// checked (us): 32 x 4096 x 4096 one part 14.2 (64 columns), two 11.2, four 10.6 (128
// columns); 64 x 1024 x 8192 27.7, 17.7, 12.5; 512 x 1024 x 8192 25.3, 17.8, 16.6;
// 256 x 4096 x 4096 15.6 whole, 15.4 and 17.2 split. Clusters of four leave SMs of a
// GPC unused (seven eighths of them are counted on); clusters of eight fit worse still
// (20 us where four took 12.5).
struct F8Shape {
  int bn, splits;
};
static F8Shape fp8_shape(int64_t row_tiles, int rows, int64_t N, int kblocks, int sms, bool may_split) {
  F8Shape best = {256, 1};
  double least = 1e30;
  const int block_ns[3] = {550, 420, 350}, quarters = (std::min(rows, kF8M) + 31) / 32;
  for (int i = 0; i < 3; ++i) {
    const int bn = 256 >> i;
    const int64_t tiles = row_tiles * ((N + bn - 1) / bn);
    for (int splits = 1; splits <= (may_split ? 4 : 1); splits *= 2) {
      if (splits > 1 && (tiles * splits > (splits == 2 ? sms : sms * 7 / 8) || splits * 2 > kblocks)) break;
      const double t = (double)((tiles * splits + sms - 1) / sms) * ((kblocks + splits - 1) / splits) * block_ns[i] +
                       (splits > 1 ? 3000 + 250 * quarters * (bn / 64) : 0);
      if (t < least) {
        least = t;
        best = {bn, splits};
      }
    }
  }
  return best;
}

template <bool GROUPED>
static mtl_status fp8_run(const char* who, const LaunchArgs& la, int M, int N, int K, int batch, int bblock, int fa, int fb,
                          int out, cudaStream_t s) {
  F8Args p = {};
  p.C = reinterpret_cast<void*>(la.a[0].ptr);
  const void* A = reinterpret_cast<const void*>(la.a[1].ptr);
  p.sA = reinterpret_cast<const float*>(la.a[2].ptr);
  const void* B = reinterpret_cast<const void*>(la.a[3].ptr);
  p.sB = reinterpret_cast<const float*>(la.a[4].ptr);
  if (GROUPED) p.offsets = reinterpret_cast<const int*>(la.a[5].ptr);
  p.M = M;
  p.N = N;
  p.K = K;
  p.batch = batch;
  p.kblocks = (K + 127) / 128;
  p.nblocks = (N + 127) / 128;
  p.vec = la.a[0].ptr % 16 == 0 && (int64_t)N * (out ? 2 : 4) % 16 == 0;
  const bool rowb = bblock == 1;
  if constexpr (!GROUPED) {
    if (M <= kFewRows && (int64_t)batch * ((N + 15) / 16) <= INT_MAX) {
      const uint8_t *a8 = static_cast<const uint8_t*>(A), *b8 = static_cast<const uint8_t*>(B);
      const cudaError_t e = M <= 8 ? (rowb ? fp8_few<1, true>(fa, fb, out, a8, b8, p, s) : fp8_few<1, false>(fa, fb, out, a8, b8, p, s))
                                   : (rowb ? fp8_few<2, true>(fa, fb, out, a8, b8, p, s) : fp8_few<2, false>(fa, fb, out, a8, b8, p, s));
      return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
  }
  p.stall = take_stall(g_fp8_stalls);  // of the kernels that wait
  if constexpr (GROUPED) {
    // Rows of a group in the MMA's N operand, 32 of them, while a group has up to 16 on
    // average and there are tiles for most SMs. Sustained, us, against tiles of 128 rows:
    // 2 rows a group (64 groups, 4096 x 2048) 89.0 and 109.4, 16 rows (2048 x 2048) 50.6
    // and 61.9, 32 rows (16 groups) 22.5 and 18.4, with 64 in the operand 18.5.
    const int64_t tiles_n = (N + 255) / 256;
    if (batch * tiles_n * 4 >= la.sm_count * 3 && M <= 16 * (int64_t)batch) {
      // 128 rows of B, kSlim rows of A; formats in that order
      p.idesc = (1u << 4) | ((uint32_t)fb << 7) | ((uint32_t)fa << 10) | ((uint32_t)(kSlim >> 3) << 17) | (8u << 24);
      CUtensorMap ta, tb;
      if (mtl_status st = make_code_map(&ta, A, K, M, 1, kSlim)) return st;
      if (mtl_status st = make_code_map(&tb, B, K, N, batch, 256)) return st;
      const int64_t tiles = ((int64_t)M / kSlim + batch) * tiles_n;
      const cudaError_t e = out ? fp8_launch_slim<kSlim, __nv_bfloat16>(ta, tb, p, tiles, la.sm_count, la.device, s)
                                : fp8_launch_slim<kSlim, float>(ta, tb, p, tiles, la.sm_count, la.device, s);
      return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
  }
  // rows a product (dense) or a group on average decide how A is loaded and how
  // many tiles there are; the groups' real sizes are on the device
  const int64_t row_tiles = GROUPED ? std::max<int64_t>(batch, (M + kF8M - 1) / kF8M) : (int64_t)((M + kF8M - 1) / kF8M) * batch;
  const F8Shape shape = fp8_shape(row_tiles, GROUPED ? M / batch : M, N, p.kblocks, la.sm_count, !GROUPED);
  const int bn = shape.bn;
  p.splits = shape.splits;
  p.a_box = (GROUPED ? M / batch : M) >= kF8M ? kF8M : 32;
  // kind::f8f6f4: fp32 accumulator (bit 4), formats at bits 7 and 10, N >> 3 at bit 17, M >> 4 at bit 24
  p.idesc = (1u << 4) | ((uint32_t)fa << 7) | ((uint32_t)fb << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(kF8M >> 4) << 24);
  CUtensorMap ta, tb;
  if (mtl_status st = make_code_map(&ta, A, K, M, GROUPED ? 1 : batch, p.a_box)) return st;
  if (mtl_status st = make_code_map(&tb, B, K, N, batch, bn)) return st;
  const int64_t tiles = (GROUPED ? (int64_t)batch + M / kF8M : row_tiles) * ((N + bn - 1) / bn);
  cudaError_t e = bn == 256   ? fp8_launch_by<256, GROUPED>(rowb, out, ta, tb, p, tiles, la.sm_count, la.device, s)
                  : bn == 128 ? fp8_launch_by<128, GROUPED>(rowb, out, ta, tb, p, tiles, la.sm_count, la.device, s)
                              : fp8_launch_by<64, GROUPED>(rowb, out, ta, tb, p, tiles, la.sm_count, la.device, s);
  return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

mtl_status gemm_fp8_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  const int M = la.a[5].i32, N = la.a[6].i32, K = la.a[7].i32, out = la.a[11].i32;
  const int64_t batch = la.nd[0];
  cudaStream_t s = (cudaStream_t)stream;
  if (batch == 0 || M == 0 || N == 0) return MTL_OK;
  if (K == 0) {  // the empty sum
    cudaError_t e = cudaMemsetAsync(reinterpret_cast<void*>(la.a[0].ptr), 0, (size_t)batch * M * N * (out ? 2 : 4), s);
    return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "gemm_fp8: %s", cudaGetErrorString(e));
  }
  return fp8_run<false>("gemm_fp8", la, M, N, K, (int)batch, la.a[8].i32, la.a[9].i32, la.a[10].i32, out, s);
}

mtl_status gemm_grouped_fp8_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  const int T = la.a[6].i32, N = la.a[7].i32, K = la.a[8].i32;
  const int64_t groups = la.nd[0];
  if (groups == 0 || T == 0 || N == 0) return MTL_OK;
  return fp8_run<true>("gemm_grouped_fp8", la, T, N, K, (int)groups, 128, la.a[9].i32, la.a[10].i32, la.a[11].i32,
                       (cudaStream_t)stream);
}

}  // namespace mtl
