// The rows of the experts back to their tokens, and the gradient.
//
//   y[t] = base[t] + sum over j of w[t, j] rows[row_at[t, j]]
//   drows[r] = w[t, j] dy[t]   dw[t, j] = <dy[t], rows[r]>   with r = row_at[t, j]
//
// Sums are 32-bit, over j in order, and y is rounded once. A slot without a row (row_at
// outside the rows there are) counts as a row of zeros. Without weights they are ones: the
// sum of a token's rows is then the gradient of gathering them, and drows the gathering.
//
// In the gradient a row is written by its own token alone, the one that rows_of names, so
// the result does not depend on timing even where two tokens name the same row; of a
// token's two slots that name one row the later counts. Rows that no slot of their token
// names are left as they were.

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "../mtl_internal.hpp"
#include "rows.cuh"

namespace mtl {

constexpr int kCombineTop = 32;

struct CombineArgs {
  void* y;
  const void* rows;
  const float* w;
  const int* row_at;
  const void* base;
  int64_t R;
  int C, top;
};

// A CTA takes a tile of a token's columns, eight a thread: B threads, or with VEC as many as make
// the tiles even.
template <typename T, typename Y, int B, bool VEC>
__global__ void __launch_bounds__(B) combine_kernel(CombineArgs a) {
  const int64_t t = blockIdx.x;
  const int tid = VEC ? blockIdx.y * blockDim.x + threadIdx.x : threadIdx.x, u = VEC ? 0 : blockIdx.y;
  const int* row_at = a.row_at + t * a.top;
  const float* weights = a.w ? a.w + t * a.top : nullptr;
  float sum[8] = {};
#pragma unroll 4
  for (int j = 0; j < a.top; ++j) {
    const int r = row_at[j];
    const float w = weights ? weights[j] : 1.0f;
    float v[8];
    if ((unsigned)r < (uint64_t)a.R) {
      load_part<B, VEC>(v, static_cast<const T*>(a.rows) + (int64_t)r * a.C, a.C, tid, u);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = fmaf(w, v[i], sum[i]);
  }
  if (a.base) {
    float v[8];
    load_part<B, VEC>(v, static_cast<const Y*>(a.base) + t * a.C, a.C, tid, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
  }
  store_part<B, VEC>(static_cast<Y*>(a.y) + t * a.C, sum, a.C, tid, u);
}

struct CombineGradArgs {
  void* drows;
  float* dw;
  const void* dy;
  const void* rows;
  const float* w;
  const int* row_at;
  const int* rows_of;
  int64_t R;
  int C, top;
};

// A CTA a token, tile by tile. WHOLE: the CTA has B threads, known when it is compiled (4096 x 2
// rows of 4096 float 56.7 -> 53.6 us, 4096 x 8 of 2048 95.8 -> 91.4; bf16 rows the same either way).
template <typename T, typename Y, int B, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(B) combine_grad_kernel(CombineGradArgs a) {
  __shared__ float part[kCombineTop][B / 32];
  const int64_t t = blockIdx.x;
  const int threads = WHOLE ? B : blockDim.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = threads >> 5, C = a.C;
  const int* row_at = a.row_at + t * a.top;
  for (int tile = 0; tile * 8 * warps * 32 < C; ++tile) {
    const int tid = VEC ? tile * threads + threadIdx.x : threadIdx.x, u = VEC ? 0 : tile;
    float g[8];
    load_part<B, VEC>(g, static_cast<const Y*>(a.dy) + t * C, C, tid, u);
#pragma unroll 4
    for (int j = 0; j < a.top; ++j) {
      const int r = row_at[j];
      const bool valid = (unsigned)r < (uint64_t)a.R;
      if (a.dw) {
        float dot = 0.0f;
        if (valid) {
          float v[8];
          load_part<B, VEC>(v, static_cast<const T*>(a.rows) + (int64_t)r * C, C, tid, u);
#pragma unroll
          for (int i = 0; i < 8; ++i) dot = fmaf(g[i], v[i], dot);
        }
        dot = warp_sum(dot);
        if (lane == 0) part[j][warp] = tile ? part[j][warp] + dot : dot;
      }
      if (valid && a.rows_of[r] == t) {
        const float w = a.w ? a.w[t * a.top + j] : 1.0f;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = w * g[i];
        store_part<B, VEC>(static_cast<T*>(a.drows) + (int64_t)r * C, d, C, tid, u);
      }
    }
  }
  if (!a.dw) return;
  __syncthreads();
  for (int j = warp; j < a.top; j += warps) {
    const float sum = warp_sum(lane < warps ? part[j][lane] : 0.0f);
    if (lane == 0) a.dw[t * a.top + j] = sum;
  }
}

// ── host side ───────────────────────────────────────────────────────────────
static mtl_status combine_sizes(const char* kernel, const LaunchArgs& la, int64_t R, int C, int top) {
  if (la.ndim != 1) return fail(MTL_ERR_ARGUMENT, "%s: ndrange must be one-dimensional (the tokens)", kernel);
  if (la.nd[0] < 0 || R < 0 || C < 0) return fail(MTL_ERR_ARGUMENT, "%s: negative dimension", kernel);
  if (top < 1 || top > kCombineTop) return fail(MTL_ERR_ARGUMENT, "%s: top must be 1 .. %d, got %d", kernel, kCombineTop, top);
  if (la.nd[0] > INT_MAX) return fail(MTL_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", kernel);
  if (C > (1 << 24)) return fail(MTL_ERR_UNSUPPORTED, "%s: more than 2^24 columns: %d", kernel, C);
  return MTL_OK;
}

// Threads of a CTA and tiles of a row, where tiles may have any size: 256 threads at most, the
// tiles even and of whole warps. Against tiles of 1024 or 2048 columns: 4000 x 2 rows of 4104
// bf16 31.2 -> 28.0 us, 8192 x 3 rows of 200 9.1 -> 6.4, their gradient 14.2 -> 10.0. Both kernels
// are bound by HBM: 8192 x 8 rows of 2048 bf16 with a base 58 us, 5.8 TB/s, the gradient 100 us,
// 5.7 TB/s. Four slots' rows loaded ahead of their sums took 70 and 170.
constexpr int kCombineThreads = 256;
struct Tiles {
  unsigned threads, tiles;
};
static Tiles even_tiles(int C) {
  const unsigned eights = (unsigned)((C + 7) / 8), tiles = (eights + kCombineThreads - 1) / kCombineThreads;
  return Tiles{((eights + tiles - 1) / tiles + 31) / 32 * 32, tiles};
}

template <typename T, typename Y>
static void combine_launch(const CombineArgs& a, int64_t tokens, bool vec, cudaStream_t st) {
  if (vec) {
    const Tiles e = even_tiles(a.C);
    combine_kernel<T, Y, kCombineThreads, true><<<dim3((unsigned)tokens, e.tiles), e.threads, 0, st>>>(a);
  } else if (a.C <= 1024) {
    combine_kernel<T, Y, 128, false><<<dim3((unsigned)tokens, 1), 128, 0, st>>>(a);
  } else {
    combine_kernel<T, Y, 256, false><<<dim3((unsigned)tokens, (unsigned)((a.C + 2047) / 2048)), 256, 0, st>>>(a);
  }
}

// Arguments: y (B), rows (B), weights (b, f32), row_at (B, i32), base (b), R, C, top, type
// of the rows (0 f32, 1 bf16), type of y and base (i); ndrange = tokens.
mtl_status combine_experts_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int64_t T = la.nd[0], R = la.a[5].i32, C = la.a[6].i32;
  const int top = la.a[7].i32;
  if (mtl_status s = combine_sizes("combine_experts", la, R, (int)C, top)) return s;
  if (mtl_status s = check_flags("combine_experts", la, {8, 9})) return s;
  const int64_t per = la.a[8].i32 ? 2 : 4, pery = la.a[9].i32 ? 2 : 4;
  const uint64_t all = bytes_of({T, C, pery}), slots = C ? bytes_of({T, top, 4}) : 0;
  return check_operands("combine_experts", la, bytes,
                        {{"y", all, (unsigned)pery},
                         {"the rows", T ? bytes_of({R, C, per}) : 0, (unsigned)per},
                         {"the weights", slots, 4},
                         {"row_at", slots, 4},
                         {"base", all, (unsigned)pery}});
}

mtl_status combine_experts_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  CombineArgs a = {};
  a.y = reinterpret_cast<void*>(la.a[0].ptr);
  a.rows = reinterpret_cast<const void*>(la.a[1].ptr);
  a.w = reinterpret_cast<const float*>(la.a[2].ptr);
  a.row_at = reinterpret_cast<const int*>(la.a[3].ptr);
  a.base = reinterpret_cast<const void*>(la.a[4].ptr);
  a.R = la.a[5].i32;
  a.C = la.a[6].i32;
  a.top = la.a[7].i32;
  const int64_t T = la.nd[0];
  if (T == 0 || a.C == 0) return MTL_OK;
  const bool vec = (la.a[0].ptr | la.a[1].ptr | la.a[4].ptr) % 16 == 0 && a.C % 8 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (la.a[8].i32)
    la.a[9].i32 ? combine_launch<uint16_t, uint16_t>(a, T, vec, st) : combine_launch<uint16_t, float>(a, T, vec, st);
  else
    la.a[9].i32 ? combine_launch<float, uint16_t>(a, T, vec, st) : combine_launch<float, float>(a, T, vec, st);
  return launched("combine_experts");
}

template <typename T, typename Y>
static void combine_grad_launch(const CombineGradArgs& a, int64_t tokens, bool vec, cudaStream_t st) {
  const unsigned grid = (unsigned)tokens;
  if (vec) {
    const unsigned threads = even_tiles(a.C).threads;
    if (threads == kCombineThreads)
      combine_grad_kernel<T, Y, kCombineThreads, true, true><<<grid, threads, 0, st>>>(a);
    else
      combine_grad_kernel<T, Y, kCombineThreads, true, false><<<grid, threads, 0, st>>>(a);
  } else if (a.C <= 1024) {
    combine_grad_kernel<T, Y, 128, false, true><<<grid, 128, 0, st>>>(a);
  } else {
    combine_grad_kernel<T, Y, 256, false, true><<<grid, 256, 0, st>>>(a);
  }
}

// Arguments: drows (B), dweights (b, f32), dy (B), rows (b), weights (b, f32), row_at (B,
// i32), rows_of (B, i32), R, C, top, type of the rows and drows, type of dy (i); ndrange =
// tokens.
mtl_status combine_experts_grad_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int64_t T = la.nd[0], R = la.a[7].i32, C = la.a[8].i32;
  const int top = la.a[9].i32;
  if (mtl_status s = combine_sizes("combine_experts_grad", la, R, (int)C, top)) return s;
  if (mtl_status s = check_flags("combine_experts_grad", la, {10, 11})) return s;
  if (given(la, 1) && !given(la, 3)) return fail(MTL_ERR_ARGUMENT, "combine_experts_grad: the weights' gradient needs the rows");
  const int64_t per = la.a[10].i32 ? 2 : 4, pery = la.a[11].i32 ? 2 : 4;
  const uint64_t all = T ? bytes_of({R, C, per}) : 0, slots = bytes_of({T, top, 4});
  return check_operands("combine_experts_grad", la, bytes,
                        {{"drows", all, (unsigned)per},
                         {"the weights' gradient", slots, 4},
                         {"dy", bytes_of({T, C, pery}), (unsigned)pery},
                         {"the rows", all, (unsigned)per},
                         {"the weights", slots, 4},
                         {"row_at", slots, 4},
                         {"rows_of", T ? bytes_of({R, 4}) : 0, 4}});
}

mtl_status combine_experts_grad_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  CombineGradArgs a = {};
  a.drows = reinterpret_cast<void*>(la.a[0].ptr);
  a.dw = reinterpret_cast<float*>(la.a[1].ptr);
  a.dy = reinterpret_cast<const void*>(la.a[2].ptr);
  a.rows = reinterpret_cast<const void*>(la.a[3].ptr);
  a.w = reinterpret_cast<const float*>(la.a[4].ptr);
  a.row_at = reinterpret_cast<const int*>(la.a[5].ptr);
  a.rows_of = reinterpret_cast<const int*>(la.a[6].ptr);
  a.R = la.a[7].i32;
  a.C = la.a[8].i32;
  a.top = la.a[9].i32;
  const int64_t T = la.nd[0];
  cudaStream_t st = (cudaStream_t)stream;
  if (T == 0) return MTL_OK;
  if (a.C == 0) {  // sums of nothing
    if (a.dw) {
      const cudaError_t e = cudaMemsetAsync(a.dw, 0, sizeof(float) * T * a.top, st);
      if (e != cudaSuccess) return fail(MTL_ERR_CUDA, "combine_experts_grad: %s", cudaGetErrorString(e));
    }
    return MTL_OK;
  }
  const bool vec = (la.a[0].ptr | la.a[2].ptr | la.a[3].ptr) % 16 == 0 && a.C % 8 == 0;
  if (la.a[10].i32)
    la.a[11].i32 ? combine_grad_launch<uint16_t, uint16_t>(a, T, vec, st) : combine_grad_launch<uint16_t, float>(a, T, vec, st);
  else
    la.a[11].i32 ? combine_grad_launch<float, uint16_t>(a, T, vec, st) : combine_grad_launch<float, float>(a, T, vec, st);
  return launched("combine_experts_grad");
}

}  // namespace mtl
