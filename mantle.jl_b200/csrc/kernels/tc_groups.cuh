// What the expert-grouped products share: the table of a launch's groups in
// shared memory and the walk of a persistent CTA over their tiles.
//
// Group e holds rows offsets[e] .. offsets[e + 1] of the row matrix. The
// offsets live on the device, so the host cannot check them: each is clamped to
// [0, rows], and one below an earlier one counts as that one. So whatever they hold,
// no access leaves the buffers, no row is in two groups, and the tiles are no more than
// the host counted.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "tc_common.cuh"

namespace mtl {

constexpr int kMaxGroups = 1024;
// The largest size of a product: the kernels round sizes and coordinates up to tiles of 256
// in 32 bits.
constexpr int kMaxSize = 0x7fffffff - 255;

struct GroupTable {
  int lo[kMaxGroups];       // first row
  int hi[kMaxGroups];       // one past the last
  int cum[kMaxGroups + 1];  // row tiles of the groups before
};

// Every thread of the CTA calls this; `tile_m` rows a tile.
__device__ __forceinline__ void build_groups(GroupTable* g, const int* __restrict__ offsets, int groups, int rows,
                                             int tile_m) {
  int falls = 0;
  for (int e = threadIdx.x; e < groups; e += blockDim.x) {
    const int lo = min(max(offsets[e], 0), rows), end = min(max(offsets[e + 1], 0), rows), hi = max(lo, end);
    falls |= end < lo;
    g->lo[e] = lo;
    g->hi[e] = hi;
    g->cum[e + 1] = (hi - lo + tile_m - 1) / tile_m;
  }
  if (__syncthreads_or(falls)) {  // not in order, which one thread mends
    if (threadIdx.x == 0) {
      int top = 0;
      for (int e = 0; e < groups; ++e) {
        g->lo[e] = top = max(top, g->lo[e]);
        g->hi[e] = max(top, g->hi[e]);
        g->cum[e + 1] = (g->hi[e] - top + tile_m - 1) / tile_m;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    int carry = 0;
    for (int base = 0; base < groups; base += 32) {
      const int e = base + (int)threadIdx.x;
      int v = e < groups ? g->cum[e + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)threadIdx.x >= d) v += u;
      }
      if (e < groups) g->cum[e + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (threadIdx.x == 0) g->cum[0] = 0;
  }
  __syncthreads();
}

// Tile t of a grouped launch, tiles in the order (group, column tile, row tile):
// neighbouring CTAs take the row tiles of one column panel of a group's weights.
// A walk asks for growing t, so the group is found by moving forward.
struct GroupWalk {
  int e = 0;
  __device__ __forceinline__ void find(const GroupTable* g, int t, int tiles_n, int tile_m, int tile_n, int* row0,
                                       int* rows, int* n0) {
    while (t >= g->cum[e + 1] * tiles_n) ++e;
    const int first = g->cum[e], mt = g->cum[e + 1] - first, in = t - first * tiles_n;
    const int m0 = in % mt * tile_m;
    *row0 = g->lo[e] + m0;
    *rows = g->hi[e] - *row0;
    *n0 = in / mt * tile_n;
  }
};

// wait_phase by a whole converged warp: the answer is the same in every lane.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort, int* timeouts) {
  bool ok = __all_sync(0xffffffffu, mbar_try_wait(bar, parity));
  if (!ok) ok = __all_sync(0xffffffffu, wait_phase(bar, parity, abort, timeouts));
  return ok;
}

// One lane of a converged warp, the choice known to the compiler to be uniform: the
// instructions behind it take their descriptors from uniform registers. Behind
// `lane == 0` four MMAs and two commits took 470 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}

// 64 or 128 bytes of each of 32 output rows, columns `col` on of `cols`, a lane holding
// its row's sums in v and `rows` rows valid: through shared memory (2 or 4 KiB of the
// warp's own), so that an instruction writes whole pieces of eight or four rows. A lane
// that stores its own row touches 32 of them with 16 bytes each: a 128 x 256 tile of fp32
// took 13000 cycles to leave that way. 128 bytes, whole lines where rows are aligned, leave
// faster where there is the room: a weight gradient that is all stores (537 MB in fp32) took
// 89 us against 115 with 64, and 102 with 128 bytes of sixteen rows at a time. 16-byte
// words are placed by word ^ row: no bank is hit twice on either side. `vec`: output rows
// start on 16 bytes.
constexpr int kStageWords = 32 * 4;  // of 64-byte pieces
template <typename OUT, int COLS>
__device__ __forceinline__ void store_rows(uint4* stage, int lane, int rows, OUT* out, int cols, int col, int vec,
                                           const float (&v)[COLS]) {
  constexpr int kPer = 16 / sizeof(OUT), kWords = COLS / kPer;  // values a word, words a row
  static_assert(kWords == 4 || kWords == 8, "64 or 128 bytes a row");
  auto at = [&](int row, int w) { return row * kWords + (w ^ (kWords == 8 ? row & 7 : row >> 1 & 3)); };
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    uint4 u;
    if constexpr (sizeof(OUT) == 4) {
      u = make_uint4(__float_as_uint(v[4 * w]), __float_as_uint(v[4 * w + 1]), __float_as_uint(v[4 * w + 2]),
                     __float_as_uint(v[4 * w + 3]));
    } else {
      __nv_bfloat162 b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[8 * w + 2 * i], v[8 * w + 2 * i + 1]);
      u = *reinterpret_cast<uint4*>(b);
    }
    stage[at(lane, w)] = u;
  }
  __syncwarp();
  if (vec) {
    const int w = lane % kWords, c = col + w * kPer;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const int row = i * (32 / kWords) + lane / kWords;
      const uint4 u = stage[at(row, w)];
      if (row < rows) {
        OUT* dst = out + (int64_t)row * cols + c;
        if (c + kPer <= cols) {
          *reinterpret_cast<uint4*>(dst) = u;
        } else {
          const OUT* e = reinterpret_cast<const OUT*>(&u);
#pragma unroll
          for (int k = 0; k < kPer; ++k)
            if (c + k < cols) dst[k] = e[k];
        }
      }
    }
  } else {
    // rows start anywhere: neighbouring lanes store neighbouring values
    constexpr int kLanes = COLS < 32 ? COLS : 32;  // lanes a row
#pragma unroll 4
    for (int row = lane / kLanes; row < 32; row += 32 / kLanes)
#pragma unroll
      for (int c = lane % kLanes; c < COLS; c += kLanes) {
        const OUT x = reinterpret_cast<const OUT*>(&stage[at(row, c / kPer)])[c % kPer];
        if (row < rows && col + c < cols) out[(int64_t)row * cols + col + c] = x;
      }
  }
  __syncwarp();
}

// ── CTA pairs ────────────────────────────────────────────────────────────────
// Two CTAs of a cluster run one tcgen05.mma (cta_group::2) on both SMs: each holds 128
// of the 256 rows of A and half of B's columns, and its tensor memory the sums of its
// rows. The even CTA issues; its barriers are reached from both through mapa. Most
// barrier operations have no .cluster scope: what they order is the async proxy's and
// tensor memory's, and a wait that acquires at cluster scope drops the L1 cache each
// time (a grouped forward product took 259 us with it, 131 without). Where a CTA stores to
// its shared memory itself, for an MMA that the even CTA issues, a release and an acquire at
// cluster scope order the two (mbar_arrive_release_cluster, mbar_acquire_cluster), restricted
// to shared memory: so they cost nothing that was measured, and whole ones, once a tile, 8 to
// 18 % (256 rows a group 140 -> 157 us).
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void mbar_expect_tx_cluster(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t bar) {
  asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// After a wait for this phase: what the threads that arrived so wrote to shared memory
// before is visible.
__device__ __forceinline__ void mbar_acquire_cluster(uint32_t bar, uint32_t parity) {
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.relaxed.cluster.shared::cta.b64 p, [%0], %1; }" ::"r"(bar), "r"(parity)
               : "memory");
  asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
}
// Loads whose barrier may be the other CTA's.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
// Arrives on the barrier at the same place in both CTAs when the MMAs so far are done.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void tc_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The MMAs in flight finish before a CTA that gives up frees its tensor memory: a whole
// converged warp calls this, for a commit covers the MMAs of the thread that makes it and
// they were issued by the lane that elect_one chooses.
template <bool PAIR>
__device__ __forceinline__ void drain_mmas(uint32_t bar) {
  if (elect_one()) {
    if (PAIR)
      tc_commit_pair(bar);
    else
      tc_commit(bar);
    drain_phase(bar, 0);
  }
  __syncwarp();
}

// Every thread of every CTA of the cluster; what each wrote to its shared memory before
// is there for the others after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// The launches left whose CTA 0 loads one K block and stops (mtl_inject_stall), so that its
// waits run out; the CTA to stop in this one, or -1.
static inline int take_stall(std::atomic<int>& launches) {
  for (int left = launches.load(std::memory_order_relaxed); left > 0;)
    if (launches.compare_exchange_weak(left, left - 1)) return 0;
  return -1;
}

// A kernel's dynamic shared memory above 48 KiB, allowed once per device.
template <typename F>
static cudaError_t allow_smem(F* kernel, int bytes, int device, unsigned long long* done) {
  if (device >= 0 && device < 64 && (__atomic_load_n(done, __ATOMIC_RELAXED) >> device & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device >= 0 && device < 64) __atomic_fetch_or(done, 1ull << device, __ATOMIC_RELAXED);
  return e;
}

}  // namespace mtl
