// Root-mean-square norm of rows, with the residual's addition before it and an output in
// 8-bit floating point behind it, and its gradient.
//
//   h = x + residual        r = 1 / sqrt(mean(h^2) + eps)        y = h r w
//
// h, the sum of squares and y are kept in 32 bits; h and y are rounded once, to x's type,
// where they are stored. The codes and scales are what quantize_fp8 makes of the 32-bit y
// in 1 x 128 blocks (definitions at the top of quantize.cu), not of its rounding to
// bfloat16. A NaN makes its row NaN, an infinity its own value NaN and the finite ones of its
// row zeros. Squares are summed in 32 bits: a row whose squares add up to more than 3.4e38, a
// mean square of 3.4e38 / C, gives zeros, and its gradient is dres alone. With eps 0 squares
// that are zeros in 32 bits (of values below 1e-23) make a row infinite, zeros a row NaN.
//
// With a = w dy and n = h r the gradient is
//
//   dx = r (a - n mean(a n)) + dres        dw = sum over rows of dy n
//
// where dres is the gradient that reaches h by the residual path. r is computed again from
// h as stored: the row is in registers anyway, and the sums of h^2 and of a h meet in one
// reduction, so the forward pass has no statistics to keep.

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "../mtl_internal.hpp"
#include "rows.cuh"
#include "tc_common.cuh"

namespace mtl {

// A row lies in the registers of one CTA, 32 values a thread at most.
constexpr int kNormColumns = 32768;

// The eights of columns that a row may touch: one more where its rows start off 16 bytes.
static int eights_of(int C) { return (C + 7) / 8 + (C % 8 && C <= kNormColumns - 8 ? 1 : 0); }
// Whether tensors whose rows start off 16 bytes are read in chunks all the same: `base` is
// their phase. (Rows of a multiple of eight that start off 16 bytes, all of them, and the
// longest rows, which the threads have no chunk more for, are read value by value.)
static bool cut_in_chunks(int C, int base) { return C % 8 ? C <= kNormColumns - 8 : base == 0; }

struct NormArgs {
  void* y;
  uint8_t* q;
  float* s;
  void* h;
  const void* x;
  const void* res;
  const void* w;
  int64_t R, Cp;
  int C, cb;
  int wbf16, e5m2, pow2;
  float eps;
};

template <int B, bool VEC>
__device__ __forceinline__ void load_weights(float (&v)[8], const void* w, int bf16, int C, int tid, int u) {
  if (bf16)
    load_part<B, VEC>(v, static_cast<const uint16_t*>(w), C, tid, u);
  else
    load_part<B, VEC>(v, static_cast<const float*>(w), C, tid, u);
}

// The sum of the row's B threads, in a fixed order. `part` holds B / 32 values.
template <int B>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = warp_sum(v);
  if constexpr (B > 32) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_sum(lane < B / 32 ? part[lane] : 0.0f);
  }
  return v;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// B threads a row: a warp each (several rows a CTA) up to 1024 columns, a CTA above; N
// eights a thread, which stay in registers between the sum and the outputs, so each value
// is read once. Bound by HBM: 8192 x 4096 bf16 with the residual, h, y and codes (303 MB)
// 49.5 us, 6.1 TB/s, 93 % of a plain copy's rate. Rows off 16 bytes are bound by the
// instructions of going value by value: 5001 x 4013 float 29 us, 5.6 TB/s, 8192 x 4095 bf16
// with the residual 63 us.
template <typename T, int B, int N, bool VEC>
__global__ void __launch_bounds__(B == 32 ? 128 : B) rms_norm_kernel(NormArgs a) {
  __shared__ float part[B == 32 ? 1 : B / 32];
  const int tid = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (B == 32 && row >= a.R) return;
  const int C = a.C;
  const int64_t at = row * C;
  float v[N][8];
#pragma unroll
  for (int u = 0; u < N; ++u) load_part<B, VEC>(v[u], static_cast<const T*>(a.x) + at, C, tid, u);
  if (a.res) {
    float o[N][8];
#pragma unroll
    for (int u = 0; u < N; ++u) load_part<B, VEC>(o[u], static_cast<const T*>(a.res) + at, C, tid, u);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] += o[u][i];
    if (a.h) {
#pragma unroll
      for (int u = 0; u < N; ++u) store_part<B, VEC>(static_cast<T*>(a.h) + at, v[u], C, tid, u);
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(v[u][i], v[u][i], sum);
  sum = row_sum<B>(sum, part);
  const float r = __frsqrt_rn(__fdiv_rn(sum, (float)C) + a.eps);
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float w[8];
    load_weights<B, VEC>(w, a.w, a.wbf16, C, tid, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[u][i] = v[u][i] * r * w[i];
    if (a.y) store_part<B, VEC>(static_cast<T*>(a.y) + at, v[u], C, tid, u);
  }
  if (!a.q) return;
  uint8_t* q = a.q + row * a.Cp;
  if constexpr (VEC) {
    // sixteen lanes a block
    const int lane16 = tid & 15;
    uint32_t m[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      m[u] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m[u] = max(m[u], magnitude(v[u][i]));
    }
    const uint32_t mine = maxima16<N>(m, lane16);
    const Scale sc = a.e5m2 ? scale_of<true>(mine, a.pow2) : scale_of<false>(mine, a.pow2);
    const int held = held_by<N>(lane16), block = (held * B + tid) >> 4;
    if (block < a.cb && lane16 == holder_of<N>(held)) a.s[(int64_t)block * a.R + row] = sc.s;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float inv = __shfl_sync(0xffffffffu, sc.r, holder_of<N>(u), 16);
      const int c = (u * B + tid) * 8;
      float2 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = mul2(make_float2(v[u][2 * i], v[u][2 * i + 1]), make_float2(inv, inv));
      const uint2 codes = a.e5m2 ? make_uint2(codes4<true>(x[0].x, x[0].y, x[1].x, x[1].y), codes4<true>(x[2].x, x[2].y, x[3].x, x[3].y))
                                 : make_uint2(codes4<false>(x[0].x, x[0].y, x[1].x, x[1].y), codes4<false>(x[2].x, x[2].y, x[3].x, x[3].y));
      // behind the row's end, up to the next row's 16 bytes, zeros
      if (c < a.Cp) *reinterpret_cast<uint2*>(q + c) = c < C ? codes : make_uint2(0, 0);
    }
  } else {
    // A block is four runs of 32 neighbouring columns, each one access of a warp. Its scale is
    // made once, and the inverse left where the maximum was.
    constexpr int kBlocks = B * N / 16;
    __shared__ uint32_t blockmax[(B == 32 ? 4 : 1) * kBlocks];
    uint32_t* most = blockmax + (B == 32 ? threadIdx.y * kBlocks : 0);
    const auto meet = [] {
      if constexpr (B == 32)
        __syncwarp();
      else
        __syncthreads();
    };
    for (int b = tid; b < kBlocks; b += B) most[b] = 0;
    meet();
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, magnitude(v[u][i]));
        if ((tid & 31) == 0) atomicMax(most + ((u * 8 + i) * B + tid) / 128, m);
      }
    meet();
    for (int b = tid; b < a.cb; b += B) {
      const Scale sc = a.e5m2 ? scale_of<true>(most[b], a.pow2) : scale_of<false>(most[b], a.pow2);
      a.s[(int64_t)b * a.R + row] = sc.s;
      most[b] = __float_as_uint(sc.r);
    }
    meet();
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = (u * 8 + i) * B + tid;
        const float x = v[u][i] * __uint_as_float(most[c / 128]);
        if (c < a.Cp) q[c] = c < C ? (uint8_t)(a.e5m2 ? codes4<true>(x, 0.0f, 0.0f, 0.0f) : codes4<false>(x, 0.0f, 0.0f, 0.0f)) : 0;
      }
  }
}

template <typename T, bool VEC>
static void norm_launch(const NormArgs& a, int sms, cudaStream_t st) {
  const unsigned rows = (unsigned)a.R, four = (unsigned)((a.R + 3) / 4);
  // Few rows: one eight a thread, so that a row takes the least time (32 x 4096 with codes
  // 3.7 -> 2.7 us, 400 x 4096 4.6 -> 4.1; 800 x 4096 6.1, and 7.5 this way).
  if (a.R < 4 * (int64_t)sms && a.C > 256 && a.C <= 8192) {
    if (a.C <= 1024)
      rms_norm_kernel<T, 128, 1, VEC><<<rows, 128, 0, st>>>(a);
    else if (a.C <= 2048)
      rms_norm_kernel<T, 256, 1, VEC><<<rows, 256, 0, st>>>(a);
    else if (a.C <= 4096)
      rms_norm_kernel<T, 512, 1, VEC><<<rows, 512, 0, st>>>(a);
    else
      rms_norm_kernel<T, 1024, 1, VEC><<<rows, 1024, 0, st>>>(a);
    return;
  }
  // Four eights a thread on 16 bytes; two off them, where four take a hundred registers and
  // leave too few threads (5001 x 4013 float 33 -> 29 us, 8192 x 4095 bf16 with the residual
  // 77 -> 63, with codes 112 -> 86; on 16 bytes two take 34 us for four's 31 of 8192 x 4096 float
  // to codes).
  if (a.C <= 256)
    rms_norm_kernel<T, 32, 1, VEC><<<four, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 512)
    rms_norm_kernel<T, 32, 2, VEC><<<four, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 1024)
    rms_norm_kernel<T, 32, 4, VEC><<<four, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 2048)
    rms_norm_kernel<T, 128, 2, VEC><<<rows, 128, 0, st>>>(a);
  else if (a.C <= 4096)
    rms_norm_kernel<T, VEC ? 128 : 256, VEC ? 4 : 2, VEC><<<rows, VEC ? 128 : 256, 0, st>>>(a);
  else if (a.C <= 8192)
    rms_norm_kernel<T, VEC ? 256 : 512, VEC ? 4 : 2, VEC><<<rows, VEC ? 256 : 512, 0, st>>>(a);
  else if (a.C <= 16384)
    rms_norm_kernel<T, 512, 4, VEC><<<rows, 512, 0, st>>>(a);
  else
    rms_norm_kernel<T, 1024, 4, VEC><<<rows, 1024, 0, st>>>(a);
}

// ── the gradient ────────────────────────────────────────────────────────────
struct NormGradArgs {
  void* dx;
  float* part;  // (gridDim.x, C) sums of dw, or null
  const void* dy;
  const void* h;
  const void* w;
  const void* dres;
  int64_t R;
  int C, wbf16, stages, base, vec;  // base: the tensors' phase; vec: they have one
  float eps;
};

// The CTAs that an SM holds: the registers are dealt out for as many, about a hundred a
// thread (at 80 the spills took 1023 x 5001 float from 20 to 22 us, 4092 rows from 48 to 61).
// So two CTAs up to 320 threads, which are 5120 columns; one of up to 640 above, and 64 registers
// beyond. The one CTA of 352 to 512 threads is the worse filled: without dres 8192 x 6144 bf16 66 us,
// 4.6 TB/s, x 8192 77 us, 5.3 TB/s; with dres, whose loads are in flight beside the others, 71.5 and
// 90 us, 5.6 and 6.0 TB/s.
constexpr int grad_residents(int most, int N) { return most == 32 ? (N == 4 ? 3 : N == 2 ? 5 : 8) : most == 128 ? 4 : most <= 320 ? 2 : 1; }
// An SM's shared memory, less what the system keeps of each CTA's (a KiB) and its static part
// (row_sums' slots, rounded up to 128 bytes), is the rings'.
constexpr size_t kRing = 204 * 1024;  // of all an SM's CTAs together
template <int MOST>
constexpr int kSumSlots = MOST == 32 ? 2 : MOST / 16;
template <int N, int MOST>
constexpr bool kRingsFit = kRing + grad_residents(MOST, N) * (1024 + (2 * kSumSlots<MOST> * sizeof(float) + 127) / 128 * 128) <= 228 * 1024;

// The sums of two values over the row's threads, in a fixed order. `part`: two slots a warp.
template <bool WARP>
__device__ __forceinline__ float2 row_sums(float x, float y, float* part) {
  const int lane = threadIdx.x & 31;
  // half the lanes go on with one value, half with the other
  float keep = lane & 16 ? y : x;
  keep += __shfl_xor_sync(0xffffffffu, lane & 16 ? x : y, 16);
#pragma unroll
  for (int d = 8; d; d >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, d);
  if constexpr (WARP) {
    return make_float2(__shfl_sync(0xffffffffu, keep, 0), __shfl_sync(0xffffffffu, keep, 16));
  } else {
    const int warps = blockDim.x >> 5;
    if ((lane & 15) == 0) part[(threadIdx.x >> 5) * 2 + (lane >> 4)] = keep;
    __syncthreads();
    float2 sum = make_float2(0.0f, 0.0f);
    const float2* p = reinterpret_cast<const float2*>(part);
    if (warps <= 8) {
      for (int w = 0; w < warps; ++w) sum.x += p[w].x, sum.y += p[w].y;
    } else {
      if (lane < warps) sum = p[lane];
      sum = make_float2(warp_sum(sum.x), warp_sum(sum.y));
    }
    return sum;
  }
}

// Bound by HBM, and by instruction issue behind that: 8192 x 4096 bf16 with dres (268 MB)
// 51 us, 5.3 TB/s, 8192 x 2048 float 47 us, 5.7 TB/s. CTAs that load, add and write in
// turn, value by value, took 95 us; with the ring and
// two values an instruction (fma.rn.f32x2) 51. Three CTAs an SM instead of two leave 80
// registers, and the spills take 60 us.
//
// CTAs stay and walk over the rows, so that a thread has the same columns in each and
// keeps their weights and their sums of dw in registers: rows that start off 16 bytes are
// taken a multiple of eight apart, whose chunks are cut alike. With RING the next rows are
// on their way into a ring of `stages` in shared memory while one is worked on; each thread
// waits for its own copies alone. Without, rows are loaded when their turn comes.
// N: its eights of values a thread.
template <typename T, int N, int MOST, bool PHASED, bool RING>
__global__ void __launch_bounds__(MOST == 32 ? 128 : MOST, grad_residents(MOST, N)) rms_norm_grad_kernel(NormGradArgs a) {
  constexpr bool WARP = MOST == 32;  // rows of a warp each
  constexpr int K = N * 8 / kWide<T>, P = kPairs<T>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) float part[2][kSumSlots<MOST>];
  const int tid = threadIdx.x, B = WARP ? 32 : blockDim.x, C = a.C;
  const int64_t stride = (int64_t)gridDim.x * blockDim.y, total = a.R * C;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int phase = PHASED && a.vec ? (int)((row * C + a.base) % (16 / (int)sizeof(T))) : 0;
  const auto chunk = [&](int u) { return chunk_of<T>(u * B + tid, phase, C); };
  pdl_trigger();  // every CTA is resident: the sums' kernel may wait beside them
  float2 dw[K][P], w[K][P];
#pragma unroll
  for (int u = 0; u < K; ++u) {
    if (a.wbf16)
      load_each(w[u], static_cast<const uint16_t*>(a.w), chunk(u), C);
    else
      load_each(w[u], static_cast<const float*>(a.w), chunk(u), C);
#pragma unroll
    for (int i = 0; i < P; ++i) dw[u][i] = make_float2(0.0f, 0.0f);
  }
  const float over = __fdiv_rn(1.0f, (float)C);
  const int image = B * K * 16, stage_bytes = image * (a.dres ? 3 : 2);
  uint8_t* mine = ring + threadIdx.y * a.stages * stage_bytes;
  const T *hs = static_cast<const T*>(a.h), *gs = static_cast<const T*>(a.dy), *ds = static_cast<const T*>(a.dres);
  const auto fetch = [&](int64_t r, int stage) {
    if constexpr (RING) {
      if (r < a.R) {
        uint8_t* to = mine + stage * stage_bytes;
#pragma unroll
        for (int u = 0; u < K; ++u) {
          const int j = u * B + tid;
          copy_chunk<PHASED>(to, j, hs, r, chunk(u), C, total);
          copy_chunk<PHASED>(to + image, j, gs, r, chunk(u), C, total);
          if (ds) copy_chunk<PHASED>(to + 2 * image, j, ds, r, chunk(u), C, total);
        }
      }
      copies_commit();
    }
  };
  for (int s = 0; s + 1 < a.stages; ++s) fetch(row + s * stride, s);
  for (int turn = 0, stage = 0; row < a.R; row += stride, turn ^= 1) {
    const uint8_t* from = mine + stage * stage_bytes;
    if constexpr (RING) copies_wait(a.stages - 2);
    const auto take = [&](float2 (&v)[P], int array, const T* p, int u) {
      if constexpr (RING)
        chunk_in<T>(v, from + array * image, u * B + tid);
      else
        load_chunk<PHASED>(v, p, row, chunk(u), C, total, a.vec);
    };
    float2 hh = make_float2(0.0f, 0.0f), ah = hh;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      float2 h[P], g[P];
      take(h, 0, hs, u);
      take(g, 1, gs, u);
      // a chunk that is partly or wholly outside the row: no part of the sums. Its later
      // values are not stored.
      if (RING && (PHASED ? chunk(u).edge : !chunk(u).on)) only_inside(h, chunk(u), C), only_inside(g, chunk(u), C);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        hh = fma2(h[i], h[i], hh);
        ah = fma2(mul2(g[i], w[u][i]), h[i], ah);
      }
      asm volatile("" ::: "memory");
    }
    // the slots are written again two rows on, behind the next row's barrier
    const float2 sums = row_sums<WARP>(hh.x + hh.y, ah.x + ah.y, part[turn]);
    // into the stage of the row before, whose last reads are behind this row's barrier
    // (or a warp's sum)
    fetch(row + (a.stages - 1) * stride, stage ? stage - 1 : a.stages - 1);
    const float r = __frsqrt_rn(sums.x * over + a.eps);
    const float2 r2 = both(r), k2 = both(-sums.y * over * r * r);
    // the row once more, from where it lies: kept in registers over the barrier it would
    // leave room for fewer threads
#pragma unroll
    for (int u = 0; u < K; ++u) {
      float2 h[P], g[P], d[P];
      take(h, 0, hs, u);
      take(g, 1, gs, u);
      if (ds) {
        take(d, 2, ds, u);
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = make_float2(0.0f, 0.0f);
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        dw[u][i] = fma2(g[i], mul2(h[i], r2), dw[u][i]);
        d[i] = fma2(r2, fma2(h[i], k2, mul2(g[i], w[u][i])), d[i]);
      }
      store_chunk<PHASED>(static_cast<T*>(a.dx), row, d, chunk(u), C, a.vec);
      asm volatile("" ::: "memory");  // one chunk after the other: the registers of one
    }
    stage = stage + 1 == a.stages ? 0 : stage + 1;
  }
  copies_wait(0);
  if (!a.part) return;
  if constexpr (WARP) {
    // The CTA's warps' sums together, each in its warp's part of the ring (two stages or more
    // of 1024 N bytes at least): as static memory they would take up to 16 KiB that the rings
    // are counted on having (two CTAs an SM instead of three at 513 to 1024 columns: 8192 x
    // 1000 bf16 20.6 us, so 16.6, 8192 x 700 float 32.6 and 21.4).
    float* meet = reinterpret_cast<float*>(ring);
    const int apart = RING ? a.stages * stage_bytes / 4 : 256 * N;
    __syncwarp();  // all lanes have read their last chunks
#pragma unroll
    for (int u = 0; u < K; ++u) {
      if (chunk(u).on) store_each(meet + threadIdx.y * apart, dw[u], chunk(u), C);
    }
    __syncthreads();
    for (int c = threadIdx.y * 32 + tid; c < C; c += 128)
      a.part[(int64_t)blockIdx.x * C + c] = meet[c] + meet[apart + c] + meet[2 * apart + c] + meet[3 * apart + c];
  } else {
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (chunk(u).on) store_each(a.part + (int64_t)blockIdx.x * C, dw[u], chunk(u), C);
  }
}

// dw = the CTAs' sums, in a fixed order: W columns a CTA, 1024 / W threads a column, each with
// every 1024 / W-th sum, eight loads in flight. 32 columns where there are many; eight, a
// sector of each sum, up to 1024 columns, whose 32 would leave most SMs idle (8192 x 200 bf16
// 10.7 -> 8.7 us, 1500 x 777 10.8 -> 9.7; 4096 x 8192 would take 47.7 us instead of 44.9).
template <int W>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(float* __restrict__ dw, const float* __restrict__ part, int parts, int C) {
  constexpr int kRows = 1024 / W;
  __shared__ float sums[W][kRows + 1];
  const int c = blockIdx.x * W + threadIdx.x;
  float sum = 0.0f;
  pdl_wait();  // the sums are the gradient kernel's
  for (int p = threadIdx.y; p < parts; p += 8 * kRows) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c < C && p + kRows * i < parts ? part[(int64_t)(p + kRows * i) * C + c] : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[i];
  }
  sums[threadIdx.x][threadIdx.y] = sum;
  __syncthreads();
  const int t = threadIdx.y * W + threadIdx.x, column = t >> 5, lane = t & 31;  // a warp a column
  if (column >= W) return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kRows / 32; ++i) sum += sums[column][lane + 32 * i];
  sum = warp_sum(sum);
  if (lane == 0 && blockIdx.x * W + column < C) dw[blockIdx.x * W + column] = sum;
}

// How a launch is laid out: CTAs of `threads` a row, `rows` rows at once a CTA, `N` eights of
// values a thread, and the ring's stages (none: rows are loaded when their turn comes, for rows
// too long for two stages).
struct GradShape {
  int threads, rows, N, most, per_sm, stages, device;
  int64_t ctas;
  size_t stage_bytes;
};
static GradShape grad_shape(int64_t R, int C, int size, bool dres, int sms) {
  GradShape g = {};
  const int eights = eights_of(C);
  g.rows = eights <= 128 ? 4 : 1;
  g.N = eights <= 32 ? 1 : eights <= 64 ? 2 : eights <= 128 ? 4 : eights <= 2048 ? 2 : 4;
  g.threads = g.rows == 4 ? 32 : (eights + 32 * g.N - 1) / (32 * g.N) * 32;
  g.most = g.threads;
  for (int most : {32, 128, 256, 320, 512, 640, 1024})
    if (g.threads <= most) {
      g.most = most;
      break;
    }
  g.per_sm = grad_residents(g.most, g.N);
  g.stage_bytes = (size_t)g.threads * g.N * 8 * size * (dres ? 3 : 2);
  while (g.per_sm > 1 && 2 * g.stage_bytes * g.rows * g.per_sm > kRing) --g.per_sm;
  g.stages = (int)std::min<size_t>(8, kRing / (g.stage_bytes * g.rows * g.per_sm));
  if (g.stages < 2) g.stages = 0;
  // no more CTAs than the turns that the longest takes need: fewer sums of dw to add up
  g.ctas = (R + g.rows - 1) / g.rows;
  const int64_t most = std::max(8, g.per_sm * sms / 8 * 8);
  if (g.ctas > most) {
    const int64_t turns = (g.ctas + most - 1) / most;
    g.ctas = ((g.ctas + turns - 1) / turns + 7) / 8 * 8;
  }
  return g;
}

template <typename T, int N, int MOST, bool PHASED, bool RING>
static cudaError_t norm_grad_go(NormGradArgs a, const GradShape& g, cudaStream_t st) {
  a.stages = RING ? g.stages : 0;
  const size_t smem = RING ? g.stage_bytes * g.rows * g.stages : MOST == 32 ? 4096 * N : 0;
  const auto kernel = rms_norm_grad_kernel<T, N, MOST, PHASED, RING>;
  if constexpr (RING) {
    static_assert(kRingsFit<N, MOST>, "an SM holds fewer CTAs than grad_shape plans");
    static unsigned long long done;
    if (const cudaError_t e = allow_shared(kernel, (int)kRing, g.device, &done)) return e;
  }
  kernel<<<(unsigned)g.ctas, dim3(g.threads, g.rows), smem, st>>>(a);
  return cudaSuccess;
}
template <typename T, bool PHASED, bool RING>
static cudaError_t norm_grad_launch(const NormGradArgs& a, const GradShape& g, cudaStream_t st) {
  if (g.rows == 4)
    return g.N == 1   ? norm_grad_go<T, 1, 32, PHASED, RING>(a, g, st)
           : g.N == 2 ? norm_grad_go<T, 2, 32, PHASED, RING>(a, g, st)
                      : norm_grad_go<T, 4, 32, PHASED, RING>(a, g, st);
  if (g.N == 4) return norm_grad_go<T, 4, 1024, PHASED, false>(a, g, st);
  if (g.most == 128) return norm_grad_go<T, 2, 128, PHASED, RING>(a, g, st);
  if (g.most == 256) return norm_grad_go<T, 2, 256, PHASED, RING>(a, g, st);
  if (g.most == 320) return norm_grad_go<T, 2, 320, PHASED, RING>(a, g, st);
  if (g.most == 512) return norm_grad_go<T, 2, 512, PHASED, RING>(a, g, st);
  if (g.most == 640) return norm_grad_go<T, 2, 640, PHASED, RING>(a, g, st);
  return norm_grad_go<T, 2, 1024, PHASED, RING>(a, g, st);
}

// ── host side ───────────────────────────────────────────────────────────────
static mtl_status norm_sizes(const char* kernel, const LaunchArgs& la, int C, float eps) {
  if (la.ndim != 1) return fail(MTL_ERR_ARGUMENT, "%s: ndrange must be one-dimensional (the rows)", kernel);
  if (C < 0 || la.nd[0] < 0) return fail(MTL_ERR_ARGUMENT, "%s: negative dimension", kernel);
  if (C > kNormColumns) return fail(MTL_ERR_UNSUPPORTED, "%s: more than %d columns: %d", kernel, kNormColumns, C);
  if (la.nd[0] > INT_MAX) return fail(MTL_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", kernel);
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(MTL_ERR_ARGUMENT, "%s: eps must be a number from 0 up, got %g", kernel, eps);
  return MTL_OK;
}

// Arguments: y (b), q (b), s (b), h (b), x (B), residual (b), w (B), C, type (0 f32, 1
// bf16; y, h, x and residual), type of w, format (0 e4m3, 1 e5m2), pow2 (i), eps (f);
// ndrange = rows.
mtl_status rms_norm_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int C = la.a[7].i32;
  if (mtl_status s = norm_sizes("rms_norm", la, C, la.a[12].f32)) return s;
  if (mtl_status s = check_flags("rms_norm", la, {8, 9, 10, 11})) return s;
  if (given(la, 1) != given(la, 2)) return fail(MTL_ERR_ARGUMENT, "rms_norm: codes and scales go together");
  if (!given(la, 0) && !given(la, 1)) return fail(MTL_ERR_ARGUMENT, "rms_norm: give y, the codes and scales, or both");
  if (given(la, 3) && !given(la, 5)) return fail(MTL_ERR_ARGUMENT, "rms_norm: without a residual h is the input itself: leave it out");
  const int64_t R = la.nd[0], per = la.a[8].i32 ? 2 : 4, perw = la.a[9].i32 ? 2 : 4;
  const unsigned al = (unsigned)per;
  const uint64_t all = bytes_of({R, C, per});
  return check_operands("rms_norm", la, bytes,
                        {{"y", all, al},
                         {"the codes", bytes_of({R, (C + 15) / 16 * 16}), 16},
                         {"the scales", bytes_of({R, (C + 127) / 128, 4}), 4},
                         {"h", all, al},
                         {"the input", all, al},
                         {"the residual", all, al},
                         {"the weights", R ? bytes_of({C, perw}) : 0, (unsigned)perw}});
}

mtl_status rms_norm_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  NormArgs a = {};
  a.y = reinterpret_cast<void*>(la.a[0].ptr);
  a.q = reinterpret_cast<uint8_t*>(la.a[1].ptr);
  a.s = reinterpret_cast<float*>(la.a[2].ptr);
  a.h = reinterpret_cast<void*>(la.a[3].ptr);
  a.x = reinterpret_cast<const void*>(la.a[4].ptr);
  a.res = reinterpret_cast<const void*>(la.a[5].ptr);
  a.w = reinterpret_cast<const void*>(la.a[6].ptr);
  a.R = la.nd[0];
  a.C = la.a[7].i32;
  if (a.R == 0 || a.C == 0) return MTL_OK;
  a.Cp = (a.C + 15) / 16 * 16;
  a.cb = (a.C + 127) / 128;
  a.wbf16 = la.a[9].i32;
  a.e5m2 = la.a[10].i32;
  a.pow2 = la.a[11].i32;
  a.eps = la.a[12].f32;
  const bool vec = (la.a[0].ptr | la.a[3].ptr | la.a[4].ptr | la.a[5].ptr | la.a[6].ptr) % 16 == 0 && a.C % 8 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (la.a[8].i32)
    vec ? norm_launch<uint16_t, true>(a, la.sm_count, st) : norm_launch<uint16_t, false>(a, la.sm_count, st);
  else
    vec ? norm_launch<float, true>(a, la.sm_count, st) : norm_launch<float, false>(a, la.sm_count, st);
  return launched("rms_norm");
}

// Arguments: dx (B), dw (b, f32), dy (B), h (B), w (B), dres (b), C, type (dx, dy, h and
// dres), type of w (i), eps (f); ndrange = rows. The scratch holds dw's partial sums.
mtl_status rms_norm_grad_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int C = la.a[6].i32;
  if (mtl_status s = norm_sizes("rms_norm_grad", la, C, la.a[9].f32)) return s;
  if (mtl_status s = check_flags("rms_norm_grad", la, {7, 8})) return s;
  const int64_t R = la.nd[0], per = la.a[7].i32 ? 2 : 4, perw = la.a[8].i32 ? 2 : 4;
  const unsigned al = (unsigned)per;
  const uint64_t all = bytes_of({R, C, per});
  return check_operands("rms_norm_grad", la, bytes,
                        {{"dx", all, al},
                         {"dw", bytes_of({C, 4}), 4},
                         {"dy", all, al},
                         {"h", all, al},
                         {"the weights", R ? bytes_of({C, perw}) : 0, (unsigned)perw},
                         {"the residual path's gradient", all, al}});
}

uint64_t rms_norm_grad_workspace(const LaunchArgs& la) {
  const int64_t R = la.nd[0], C = la.a[6].i32;
  if (la.a[1].kind != MTL_ARG_PTR || R <= 0 || C <= 0 || C > kNormColumns) return 0;
  return bytes_of({grad_shape(R, (int)C, la.a[7].i32 ? 2 : 4, given(la, 5), la.sm_count).ctas, C, 4});
}

mtl_status rms_norm_grad_run(const LaunchArgs& la, void* ws, uint64_t ws_bytes, void* stream) {
  NormGradArgs a = {};
  a.dx = reinterpret_cast<void*>(la.a[0].ptr);
  float* dw = reinterpret_cast<float*>(la.a[1].ptr);
  a.dy = reinterpret_cast<const void*>(la.a[2].ptr);
  a.h = reinterpret_cast<const void*>(la.a[3].ptr);
  a.w = reinterpret_cast<const void*>(la.a[4].ptr);
  a.dres = reinterpret_cast<const void*>(la.a[5].ptr);
  a.R = la.nd[0];
  a.C = la.a[6].i32;
  a.wbf16 = la.a[8].i32;
  a.eps = la.a[9].f32;
  if (a.C == 0) return MTL_OK;
  cudaStream_t st = (cudaStream_t)stream;
  const uint64_t need = rms_norm_grad_workspace(la);
  if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
    return fail(MTL_ERR_ARGUMENT, "rms_norm_grad: dw needs %llu bytes of scratch on 16 bytes (mtl_kernel_workspace), got %llu",
                (unsigned long long)need, (unsigned long long)(ws ? ws_bytes : 0));
  a.part = dw ? static_cast<float*>(ws) : nullptr;
  const bool bf16 = la.a[7].i32;
  const int size = bf16 ? 2 : 4;
  a.base = phase_of(la.a[0].ptr, size);
  a.vec = cut_in_chunks(a.C, a.base);
  for (int i : {2, 3, 5}) a.vec &= !given(la, i) || phase_of(la.a[i].ptr, size) == a.base;
  GradShape g = grad_shape(a.R, a.C, size, given(la, 5), la.sm_count);
  g.device = la.device;
  const bool phased = !a.vec || a.C % 8, ring = a.vec && g.stages;
  if (a.R) {
    cudaError_t e;
    if (bf16)
      e = !phased ? (ring ? norm_grad_launch<uint16_t, false, true>(a, g, st) : norm_grad_launch<uint16_t, false, false>(a, g, st))
                  : (ring ? norm_grad_launch<uint16_t, true, true>(a, g, st) : norm_grad_launch<uint16_t, true, false>(a, g, st));
    else
      e = !phased ? (ring ? norm_grad_launch<float, false, true>(a, g, st) : norm_grad_launch<float, false, false>(a, g, st))
                  : (ring ? norm_grad_launch<float, true, true>(a, g, st) : norm_grad_launch<float, true, false>(a, g, st));
    if (e != cudaSuccess) return fail(MTL_ERR_CUDA, "rms_norm_grad: %s", cudaGetErrorString(e));
  }
  if (dw) {
    const float* sums = a.part;
    const cudaError_t e = a.C <= 1024 ? launch_pdl(rms_norm_dw_kernel<8>, dim3((a.C + 7) / 8), dim3(8, 128), 0, st, dw, sums, (int)g.ctas, a.C)
                                      : launch_pdl(rms_norm_dw_kernel<32>, dim3((a.C + 31) / 32), dim3(32, 32), 0, st, dw, sums, (int)g.ctas, a.C);
    if (e != cudaSuccess) return fail(MTL_ERR_CUDA, "rms_norm_grad: %s", cudaGetErrorString(e));
  }
  return launched("rms_norm_grad");
}

}  // namespace mtl
