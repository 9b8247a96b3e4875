// Root-mean-square norm of rows, with the residual's addition before it and an output in
// 8-bit floating point behind it, and its gradient.
//
//   h = x + residual        r = 1 / sqrt(mean(h^2) + eps)        y = h r w
//
// h, the sum of squares and y are kept in 32 bits; h and y are rounded once, to x's type,
// where they are stored. The codes and scales are what quantize_fp8 makes of the 32-bit y
// in 1 x 128 blocks (definitions at the top of quantize.cu), not of its rounding to
// bfloat16. A NaN or an infinity makes its row NaN. Squares are summed in 32 bits, so a row
// whose mean square passes 3.4e38 gives zeros.
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

namespace mtl {

// A row lies in the registers of one CTA, 32 values a thread at most.
constexpr int kNormColumns = 32768;

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

// B threads a row: a warp each (several rows a CTA) up to 1024 columns, a CTA above.
template <typename T, int B, int N, bool VEC>
__global__ void __launch_bounds__(B == 32 ? 128 : B) rms_norm_kernel(NormArgs a) {
  __shared__ float part[B == 32 ? 1 : B / 32];
  __shared__ uint32_t blockmax[VEC ? 1 : B == 32 ? 4 * 2 * N : B * N / 16];
  const int tid = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (B == 32 && row >= a.R) return;
  const int C = a.C;
  const int64_t at = row * C;
  float v[N][8];
  load_row<B, N, VEC>(v, static_cast<const T*>(a.x) + at, C, tid);
  if (a.res) {
    float o[N][8];
    load_row<B, N, VEC>(o, static_cast<const T*>(a.res) + at, C, tid);
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
    // a block is four runs of 32 neighbouring columns, each one access of a warp
    uint32_t* most = B == 32 ? blockmax + threadIdx.y * 2 * N : blockmax;
    constexpr int kBlocks = B * N / 16;
    for (int b = tid; b < kBlocks; b += B) most[b] = 0;
    if constexpr (B == 32)
      __syncwarp();
    else
      __syncthreads();
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, magnitude(v[u][i]));
        if ((tid & 31) == 0) atomicMax(most + ((u * 8 + i) * B + tid) / 128, m);
      }
    if constexpr (B == 32)
      __syncwarp();
    else
      __syncthreads();
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = (u * 8 + i) * B + tid;
        if (c >= a.Cp) continue;
        const Scale sc = a.e5m2 ? scale_of<true>(most[c / 128], a.pow2) : scale_of<false>(most[c / 128], a.pow2);
        if (c % 128 == 0 && c < C) a.s[(int64_t)(c / 128) * a.R + row] = sc.s;
        const float x = v[u][i] * sc.r;
        q[c] = c < C ? (uint8_t)(a.e5m2 ? codes4<true>(x, 0.0f, 0.0f, 0.0f) : codes4<false>(x, 0.0f, 0.0f, 0.0f)) : 0;
      }
  }
}

template <typename T, bool VEC>
static void norm_launch(const NormArgs& a, cudaStream_t st) {
  const unsigned rows = (unsigned)a.R, four = (unsigned)((a.R + 3) / 4);
  if (a.C <= 256)
    rms_norm_kernel<T, 32, 1, VEC><<<four, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 512)
    rms_norm_kernel<T, 32, 2, VEC><<<four, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 1024)
    rms_norm_kernel<T, 32, 4, VEC><<<four, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 2048)
    rms_norm_kernel<T, 128, 2, VEC><<<rows, 128, 0, st>>>(a);
  else if (a.C <= 4096)
    rms_norm_kernel<T, 128, 4, VEC><<<rows, 128, 0, st>>>(a);
  else if (a.C <= 8192)
    rms_norm_kernel<T, 256, 4, VEC><<<rows, 256, 0, st>>>(a);
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
  int C, wbf16;
  float eps;
};

// CTAs stay and walk over the rows, so that a thread has the same columns in each and
// keeps their sums of dw in registers.
template <typename T, int B, int N, bool VEC>
__global__ void __launch_bounds__(B == 32 ? 128 : B) rms_norm_grad_kernel(NormGradArgs a) {
  __shared__ float part[2][2][B == 32 ? 1 : B / 32];
  __shared__ float meet[B == 32 ? 4 * 256 * N : 1];
  const int tid = threadIdx.x, C = a.C;
  float dw[N][8];
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[u][i] = 0.0f;
  int turn = 0;
  const float over = __fdiv_rn(1.0f, (float)C);
  for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < a.R; row += (int64_t)gridDim.x * blockDim.y, turn ^= 1) {
    const int64_t at = row * C;
    float h[N][8], g[N][8];
    load_row<B, N, VEC>(h, static_cast<const T*>(a.h) + at, C, tid);
    load_row<B, N, VEC>(g, static_cast<const T*>(a.dy) + at, C, tid);
    float hh = 0.0f, ah = 0.0f;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float w[8];
      load_weights<B, VEC>(w, a.w, a.wbf16, C, tid, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hh = fmaf(h[u][i], h[u][i], hh);
        ah = fmaf(g[u][i] * w[i], h[u][i], ah);
      }
    }
    hh = warp_sum(hh);
    ah = warp_sum(ah);
    if constexpr (B > 32) {
      // written again two rows on, behind the next row's barrier
      const int lane = tid & 31;
      if (lane == 0) part[turn][0][tid >> 5] = hh, part[turn][1][tid >> 5] = ah;
      __syncthreads();
      hh = warp_sum(lane < B / 32 ? part[turn][0][lane] : 0.0f);
      ah = warp_sum(lane < B / 32 ? part[turn][1][lane] : 0.0f);
    }
    const float r = __frsqrt_rn(hh * over + a.eps), k = ah * over * r * r;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float w[8], d[8];
      load_weights<B, VEC>(w, a.w, a.wbf16, C, tid, u);
      if (a.dres) {
        load_part<B, VEC>(d, static_cast<const T*>(a.dres) + at, C, tid, u);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[u][i] = fmaf(g[u][i], h[u][i] * r, dw[u][i]);
        d[i] = fmaf(r, fmaf(-h[u][i], k, g[u][i] * w[i]), d[i]);
      }
      store_part<B, VEC>(static_cast<T*>(a.dx) + at, d, C, tid, u);
    }
  }
  if (!a.part) return;
  if constexpr (B == 32) {  // the CTA's warps' sums together
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) meet[threadIdx.y * 256 * N + (u * 8 + i) * 32 + tid] = dw[u][i];
    __syncthreads();
    if (threadIdx.y) return;
    for (unsigned y = 1; y < blockDim.y; ++y)
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[u][i] += meet[y * 256 * N + (u * 8 + i) * 32 + tid];
  }
#pragma unroll
  for (int u = 0; u < N; ++u) store_part<B, VEC>(a.part + (int64_t)blockIdx.x * C, dw[u], C, tid, u);
}

// dw = the CTAs' sums, in their order: 32 columns a CTA, sixteen threads a column.
__global__ void __launch_bounds__(512) rms_norm_dw_kernel(float* __restrict__ dw, const float* __restrict__ part, int parts, int C) {
  __shared__ float sums[16][32];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.0f;
  if (c < C)
    for (int p = threadIdx.y; p < parts; p += 16) sum += part[(int64_t)p * C + c];
  sums[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    for (int y = 1; y < 16; ++y) sum += sums[y][threadIdx.x];
    dw[c] = sum;
  }
}

// The CTAs of a launch: what an SM holds of them, and no more than there are rows.
static int64_t grad_ctas(int64_t R, int C, int sms) {
  if (C <= 1024) return std::min<int64_t>((R + 3) / 4, 4 * (int64_t)sms);
  return std::min<int64_t>(R, (C <= 4096 ? 4 : C <= 8192 ? 2 : 1) * (int64_t)sms);
}

template <typename T, bool VEC>
static void norm_grad_launch(const NormGradArgs& a, unsigned ctas, cudaStream_t st) {
  if (a.C <= 256)
    rms_norm_grad_kernel<T, 32, 1, VEC><<<ctas, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 512)
    rms_norm_grad_kernel<T, 32, 2, VEC><<<ctas, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 1024)
    rms_norm_grad_kernel<T, 32, 4, VEC><<<ctas, dim3(32, 4), 0, st>>>(a);
  else if (a.C <= 2048)
    rms_norm_grad_kernel<T, 128, 2, VEC><<<ctas, 128, 0, st>>>(a);
  else if (a.C <= 4096)
    rms_norm_grad_kernel<T, 256, 2, VEC><<<ctas, 256, 0, st>>>(a);
  else if (a.C <= 8192)
    rms_norm_grad_kernel<T, 512, 2, VEC><<<ctas, 512, 0, st>>>(a);
  else if (a.C <= 16384)
    rms_norm_grad_kernel<T, 1024, 2, VEC><<<ctas, 1024, 0, st>>>(a);
  else
    rms_norm_grad_kernel<T, 1024, 4, VEC><<<ctas, 1024, 0, st>>>(a);
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
    vec ? norm_launch<uint16_t, true>(a, st) : norm_launch<uint16_t, false>(a, st);
  else
    vec ? norm_launch<float, true>(a, st) : norm_launch<float, false>(a, st);
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
  return bytes_of({grad_ctas(R, (int)C, la.sm_count), C, 4});
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
  const int ctas = a.R ? (int)grad_ctas(a.R, a.C, la.sm_count) : 0;
  a.part = dw ? static_cast<float*>(ws) : nullptr;
  const bool vec = (la.a[0].ptr | la.a[2].ptr | la.a[3].ptr | la.a[4].ptr | la.a[5].ptr) % 16 == 0 && a.C % 8 == 0;
  if (ctas) {
    if (la.a[7].i32)
      vec ? norm_grad_launch<uint16_t, true>(a, ctas, st) : norm_grad_launch<uint16_t, false>(a, ctas, st);
    else
      vec ? norm_grad_launch<float, true>(a, ctas, st) : norm_grad_launch<float, false>(a, ctas, st);
  }
  if (dw) rms_norm_dw_kernel<<<(a.C + 31) / 32, dim3(32, 16), 0, st>>>(dw, a.part, ctas, a.C);
  return launched("rms_norm_grad");
}

}  // namespace mtl
