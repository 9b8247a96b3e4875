// Values to 8-bit floating point in blocks of 128 with one scale a block, the
// operands of gemm_fp8 and gemm_grouped_fp8.
//
// With a the largest magnitude in the block, but at least 2^-96, and L the
// format's largest value (448 for e4m3, 57344 for e5m2):
//
//   scale = fl32(a / L)    r = fl32(L / a)    code = round8(fl32(x * r))
//
// rounded to the nearest, ties to even; |x * r| exceeds L by one unit of fp32 at
// most, which rounds back to L. With pow2 the scale is the smallest power of two
// s with a <= L * s and r = 1 / s, so both products are exact. The floor keeps
// r finite and gives a block of zeros a scale that can be divided by. A NaN in
// a block makes its scale and all its codes NaN (the largest magnitude is found
// on the bits, where NaN is above infinity); an infinity makes the scale
// infinite, itself NaN and the finite values 0.
//
// A block is 1 x 128 along a row or a 128 x 128 square. The transposed outputs
// are what the input's transpose would give: for a row block, columns in runs of
// 128 rows. Rows of codes start every 16 bytes rounded up (TMA's row stride) and
// the bytes between are zeros.
//
// A value is read once, kept in registers, and written once per output, so that HBM is
// the bound to reach; the figures are at each kernel (a device-to-device copy reaches
// 5.4 TB/s at these sizes).

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "../mtl_internal.hpp"

namespace mtl {

struct QuantArgs {
  uint8_t* q;         // R rows of Cp codes, or null
  float* s;
  uint8_t* qt;        // C rows of Rp codes, or null
  float* st;
  const void* x;
  const int* rows_of;  // source row of each row, or null
  int64_t R, C, Cp, Rp;
  int64_t rb, cb;      // blocks of 128 rows / columns
  int xrows;           // rows of x that rows_of may name
  int pow2, vec;  // vec: every row of x starts on 16 bytes
};

// ── values ──────────────────────────────────────────────────────────────────
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }

// Eight neighbouring values as loaded, zeros from column C on.
template <typename T>
struct Raw8;
template <>
struct Raw8<uint16_t> {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const uint16_t* row, int64_t c, int64_t C, int vec) {
    if (vec && c + 8 <= C) {
      u = __ldg(reinterpret_cast<const uint4*>(row + c));
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = c + i < C ? row[c + i] : 0;
      u = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
  }
  // magnitudes, two to a word: m[i] = max(m[i], |values 2 i and 2 i + 1|)
  static constexpr int kWords = 4;
  __device__ __forceinline__ uint32_t mag(int i) const { return (i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w) & 0x7fff7fffu; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  // the fp32 bits of column c's magnitude, and of the largest in a word
  static __device__ __forceinline__ uint32_t column(const uint32_t (&m)[4], int c) { return c & 1 ? m[c / 2] & 0xffff0000u : m[c / 2] << 16; }
  static __device__ __forceinline__ uint32_t whole(uint32_t m) { return max(m & 0xffff0000u, m << 16); }
  __device__ __forceinline__ float2 pair(int i) const {  // values 2 i and 2 i + 1
    const uint32_t w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
    return make_float2(bf16_lo(w), bf16_hi(w));
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const float* row, int64_t c, int64_t C, int vec) {
    if (vec && c + 8 <= C) {
      a = __ldg(reinterpret_cast<const float4*>(row + c));
      b = __ldg(reinterpret_cast<const float4*>(row + c + 4));
    } else {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = c + i < C ? row[c + i] : 0.0f;
      a = make_float4(w[0], w[1], w[2], w[3]);
      b = make_float4(w[4], w[5], w[6], w[7]);
    }
  }
  static constexpr int kWords = 8;
  __device__ __forceinline__ uint32_t mag(int i) const {
    const float2 p = pair(i / 2);
    return __float_as_uint(i & 1 ? p.y : p.x) & 0x7fffffffu;
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t column(const uint32_t (&m)[8], int c) { return m[c]; }
  static __device__ __forceinline__ uint32_t whole(uint32_t m) { return m; }
  __device__ __forceinline__ float2 pair(int i) const {
    return i == 0 ? make_float2(a.x, a.y) : i == 1 ? make_float2(a.z, a.w) : i == 2 ? make_float2(b.x, b.y) : make_float2(b.z, b.w);
  }
};

// The input row behind output row r: null where it is past the end or rows_of
// names none (its values are then zeros).
template <typename T>
__device__ __forceinline__ const T* source_row(const QuantArgs& a, int64_t batch, int64_t r) {
  if (r >= a.R) return nullptr;
  const T* x = static_cast<const T*>(a.x);
  if (a.rows_of) {
    const int from = a.rows_of[r];
    return from >= 0 && from < a.xrows ? x + (int64_t)from * a.C : nullptr;
  }
  return x + (batch * a.R + r) * a.C;
}

struct Scale {
  float s, r;
};
template <bool E5M2>
__device__ __forceinline__ Scale scale_of(uint32_t bits, int pow2) {
  bits = max(bits, (uint32_t)(127 - 96) << 23);
  const float a = __uint_as_float(bits), top = E5M2 ? 57344.0f : 448.0f;
  if (pow2 && bits < 0x7f800000u) {
    // a = m 2^e, m in [1, 2), and L = 1.75 2^8 or 1.75 2^15
    const int j = (int)(bits >> 23) - 127 - (E5M2 ? 15 : 8) + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return Scale{__uint_as_float((uint32_t)(127 + j) << 23), __uint_as_float((uint32_t)(127 - j) << 23)};
  }
  return Scale{__fdiv_rn(a, top), __fdiv_rn(top, a)};
}

// Four codes, the first in the low byte.
template <bool E5M2>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  uint32_t u;
  if constexpr (E5M2)
    asm("{ .reg .b16 l, h; cvt.rn.satfinite.e5m2x2.f32 l, %2, %1; cvt.rn.satfinite.e5m2x2.f32 h, %4, %3; mov.b32 %0, {l, h}; }"
        : "=r"(u)
        : "f"(a), "f"(b), "f"(c), "f"(d));
  else
    asm("{ .reg .b16 l, h; cvt.rn.satfinite.e4m3x2.f32 l, %2, %1; cvt.rn.satfinite.e4m3x2.f32 h, %4, %3; mov.b32 %0, {l, h}; }"
        : "=r"(u)
        : "f"(a), "f"(b), "f"(c), "f"(d));
  return u;
}
// Two products an instruction, each rounded to the nearest as one alone is.
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
  float2 z;
  asm("{ .reg .b64 a, b; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 a, a, b; mov.b64 {%0, %1}, a; }"
      : "=f"(z.x), "=f"(z.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return z;
}
template <bool E5M2, typename RAW>
__device__ __forceinline__ uint2 codes8(const RAW& v, float r) {  // of a row
  float2 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = mul2(v.pair(i), make_float2(r, r));
  return make_uint2(codes4<E5M2>(x[0].x, x[0].y, x[1].x, x[1].y), codes4<E5M2>(x[2].x, x[2].y, x[3].x, x[3].y));
}

// What lies between rows of codes is zeros times an inverse, so zeros but where the inverse
// is NaN. There the thread that wrote the eight codes at `at` of a row clears those that are
// not below `end`, the row's length; with a test in every write 8192 x 4096 rows took 18.2 us
// instead of 17.2.
__device__ __forceinline__ void clear_padding(uint8_t* codes, int64_t at, int64_t end) {
  for (int64_t i = at > end ? at : end; i < at + 8; ++i) codes[i - at] = 0;
}

// The maxima of N values over 16 lanes at once: a step halves the values a lane
// keeps, so N values take N + log2(16 / N) shuffles where N separate reductions take
// 4 N, and each lane ends with one value's maximum: value held_by(lane). The two
// divisions of a scale are then one lane's, and its inverse goes back by a shuffle.
template <int N>
__device__ __forceinline__ uint32_t maxima16(uint32_t (&v)[N], int lane16) {
  int d = 8;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2, d /= 2) {
    const bool up = lane16 & d;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const uint32_t mine = up ? v[i + n] : v[i], other = up ? v[i] : v[i + n];
      v[i] = max(mine, __shfl_xor_sync(0xffffffffu, other, d));
    }
  }
  uint32_t m = v[0];
#pragma unroll
  for (; d >= 1; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}
template <int N>
__device__ __forceinline__ int held_by(int lane16) {  // value lane16 holds
  return lane16 / (16 / N);
}
template <int N>
__device__ __forceinline__ int holder_of(int value) {  // the first lane that holds it
  return value * (16 / N);
}

// ── row blocks, no transpose ────────────────────────────────────────────────
// Sixteen lanes a block of 128 (eight values each), a CTA sixteen rows of U
// neighbouring blocks: the U loads of a thread are in flight together, and the
// scales of sixteen rows leave as one 64-byte run. 8192 x 4096 bf16: 18.1 us, 5.6 TB/s
// (26 with the two divisions of a scale in every lane). Rows that do not start on 16
// bytes are loaded value by value: 8192 x 4095 30.5 us; aligned words around them,
// shifted into place, took 28.6, and in fp32 38.7 instead of 36.3.
constexpr int kQuantThreads = 256;
template <typename T, int U, bool E5M2>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 2 ? 6 : 4) quantize_rows_kernel(QuantArgs a, unsigned row_tiles, unsigned col_tiles) {
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const unsigned b = blockIdx.x / (row_tiles * col_tiles), in = blockIdx.x % (row_tiles * col_tiles);
  const int64_t batch = b, r = in / col_tiles * 16 + sub, kb0 = in % col_tiles * U;
  const T* row = source_row<T>(a, batch, r);
  Raw8<T> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    raw[u].zero();
    if (row) raw[u].load(row, (kb0 + u) * 128 + lane16 * 8, a.C, a.vec);
  }
  uint32_t m[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t w = raw[u].mag(0);
#pragma unroll
    for (int i = 1; i < Raw8<T>::kWords; ++i) w = Raw8<T>::larger(w, raw[u].mag(i));
    m[u] = Raw8<T>::whole(w);
  }
  const Scale sc = scale_of<E5M2>(maxima16<U>(m, lane16), a.pow2);
  const int64_t mine = kb0 + held_by<U>(lane16);
  if (r < a.R && mine < a.cb && lane16 == holder_of<U>(held_by<U>(lane16))) a.s[(batch * a.cb + mine) * a.R + r] = sc.s;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv = __shfl_sync(0xffffffffu, sc.r, holder_of<U>(u), 16);
    const int64_t c = (kb0 + u) * 128 + lane16 * 8;
    if (r < a.R && c < a.Cp)
      *reinterpret_cast<uint2*>(a.q + (batch * a.R + r) * a.Cp + c) = codes8<E5M2>(raw[u], inv);
  }
  if (__any_sync(0xffffffffu, isnan(sc.r)))
    for (int u = 0; u < U; ++u) {
      const int64_t c = (kb0 + u) * 128 + lane16 * 8;
      if (r < a.R && c < a.Cp) clear_padding(a.q + (batch * a.R + r) * a.Cp + c, c, a.C);
    }
}

// ── 128 x 128 tiles: square blocks, transposed outputs ──────────────────────
// A thread holds an 8 x 8 patch (eight rows of eight columns), so it can pack
// eight codes along a row and eight down a column. Row maxima meet over the
// sixteen lanes of a row, column maxima over the CTA through shared memory. The
// transposed codes go through a 16 KiB tile whose 8-byte chunks are placed by
// chunk ^ (column / 8): the sixteen lanes that write one instruction's columns
// hit all 32 banks, and so do the sixteen that read a transposed row. 8192 x 4096 bf16
// both ways: 29.9 us, 4.6 TB/s (52 with the scales' divisions in every lane and 64-bit
// tile indexes, 35 with magnitudes compared one by one; 33 at three CTAs an SM); a
// thousand rows more take 3.03 us, 5.5 TB/s and so the copy's rate, and 5 us are the
// launch and the first and last tiles' time. 5001 x 4100 fp32 in squares 25.3 us, 4.8 TB/s.
template <typename T, bool E5M2>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 2 ? 4 : 3) quantize_tile_kernel(QuantArgs a, int square) {
  __shared__ alignas(16) uint32_t colmax[8][128];
  __shared__ uint2 turned[128 * 16];
  __shared__ alignas(8) float inv[128];
  __shared__ uint32_t tilemax[8];
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const unsigned cb = (unsigned)a.cb, tiles = (unsigned)a.rb * cb, b = blockIdx.x / tiles, in = blockIdx.x % tiles;
  const int64_t batch = b, rblk = in / cb, kb = in % cb;
  const int64_t r0 = rblk * 128 + sub * 8, c = kb * 128 + lane16 * 8;
  Raw8<T> raw[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const T* row = source_row<T>(a, batch, r0 + p);
    raw[p].zero();
    if (row) raw[p].load(row, c, a.C, a.vec);
  }
  using Raw = Raw8<T>;
  uint32_t cm[Raw::kWords], rm[8];
#pragma unroll
  for (int i = 0; i < Raw::kWords; ++i) cm[i] = 0;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    uint32_t row = 0;
#pragma unroll
    for (int i = 0; i < Raw::kWords; ++i) {
      const uint32_t m = raw[p].mag(i);
      row = Raw::larger(row, m);
      cm[i] = Raw::larger(cm[i], m);
    }
    rm[p] = Raw::whole(row);
  }
  bool bad = false;  // an inverse is NaN: there is a NaN in the tile, so one of a row and one of a column are
  auto clear_rows = [&]() {
#pragma unroll 1
    for (int p = 0; p < 8; ++p)
      if (r0 + p < a.R && c < a.Cp) clear_padding(a.q + (batch * a.R + r0 + p) * a.Cp + c, c, a.C);
  };
  if (square) {
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) m = max(m, rm[p]);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) tilemax[warp] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, tilemax[w]);
    const Scale sc = scale_of<E5M2>(m, a.pow2);
    if (threadIdx.x == 0) {
      if (a.s) a.s[(batch * a.rb + rblk) * a.cb + kb] = sc.s;
      if (a.st) a.st[(batch * a.cb + kb) * a.rb + rblk] = sc.s;
    }
    if (a.q) {
#pragma unroll
      for (int p = 0; p < 8; ++p)
        if (r0 + p < a.R && c < a.Cp)
          *reinterpret_cast<uint2*>(a.q + (batch * a.R + r0 + p) * a.Cp + c) = codes8<E5M2>(raw[p], sc.r);
    }
    bad = isnan(sc.r);
    if (!a.qt) {  // row blocks alone are the other kernel's
      if (bad) clear_rows();
      return;
    }
    if (threadIdx.x < 128) inv[threadIdx.x] = sc.r;
  } else {
    if (a.q) {
      const Scale sc = scale_of<E5M2>(maxima16<8>(rm, lane16), a.pow2);
      const int64_t mine = r0 + held_by<8>(lane16);
      if (mine < a.R && (lane16 & 1) == 0) a.s[(batch * a.cb + kb) * a.R + mine] = sc.s;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float rinv = __shfl_sync(0xffffffffu, sc.r, holder_of<8>(p), 16);
        if (r0 + p < a.R && c < a.Cp)
          *reinterpret_cast<uint2*>(a.q + (batch * a.R + r0 + p) * a.Cp + c) = codes8<E5M2>(raw[p], rinv);
      }
    }
#pragma unroll
    for (int i = 0; i < Raw::kWords; ++i) cm[i] = Raw::larger(cm[i], __shfl_xor_sync(0xffffffffu, cm[i], 16));
    if ((threadIdx.x & 31) < 16) {
#pragma unroll
      for (int i = 0; i < 8; i += 4)
        *reinterpret_cast<uint4*>(&colmax[warp][lane16 * 8 + i]) =
            make_uint4(Raw::column(cm, i), Raw::column(cm, i + 1), Raw::column(cm, i + 2), Raw::column(cm, i + 3));
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) m = max(m, colmax[w][threadIdx.x]);
      const Scale sc = scale_of<E5M2>(m, a.pow2);
      inv[threadIdx.x] = sc.r;
      bad = isnan(sc.r);
      const int64_t col = kb * 128 + threadIdx.x;
      if (col < a.C) a.st[(batch * a.rb + rblk) * a.C + col] = sc.s;
    }
  }
  bad = __syncthreads_or(bad);
  // columns as rows: eight codes down each of the thread's eight columns, two columns at once
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 r = *reinterpret_cast<const float2*>(&inv[lane16 * 8 + 2 * i]);
    float2 x[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) x[p] = mul2(raw[p].pair(i), r);
    uint2* to = &turned[(lane16 * 8 + 2 * i) * 16 + (sub ^ lane16)];
    to[0] = make_uint2(codes4<E5M2>(x[0].x, x[1].x, x[2].x, x[3].x), codes4<E5M2>(x[4].x, x[5].x, x[6].x, x[7].x));
    to[16] = make_uint2(codes4<E5M2>(x[0].y, x[1].y, x[2].y, x[3].y), codes4<E5M2>(x[4].y, x[5].y, x[6].y, x[7].y));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int col = sub * 8 + i;  // sixteen lanes write one transposed row's 128 bytes
    const int64_t at = rblk * 128 + lane16 * 8;
    if (kb * 128 + col < a.C && at < a.Rp)
      *reinterpret_cast<uint2*>(a.qt + (batch * a.C + kb * 128 + col) * a.Rp + at) = turned[col * 16 + (lane16 ^ sub)];
  }
  if (bad) {
    if (a.q) clear_rows();
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const int64_t col = kb * 128 + sub * 8 + i, at = rblk * 128 + lane16 * 8;
      if (col < a.C && at < a.Rp) clear_padding(a.qt + (batch * a.C + col) * a.Rp + at, at, a.R);
    }
  }
}

// ── host side ───────────────────────────────────────────────────────────────
// Arguments: q (b), s (b), qt (b), st (b), x (B), rows_of (b, i32), R, C, xrows,
// block, type (0 f32, 1 bf16), format (0 e4m3, 1 e5m2), pow2 (i); ndrange = batch.
static int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

mtl_status quantize_check(const LaunchArgs& la, const uint64_t* bytes) {
  if (la.ndim != 1) return fail(MTL_ERR_ARGUMENT, "quantize_fp8: ndrange must be one-dimensional (the batch count)");
  const int64_t R = la.a[6].i32, C = la.a[7].i32, xrows = la.a[8].i32, batch = la.nd[0];
  const int block = la.a[9].i32;
  if (R < 0 || C < 0 || xrows < 0) return fail(MTL_ERR_ARGUMENT, "quantize_fp8: negative dimension");
  if (block != 1 && block != 128)
    return fail(MTL_ERR_ARGUMENT, "quantize_fp8: block must be 1 (1 x 128) or 128 (128 x 128), got %d", block);
  for (int i = 10; i < 13; ++i)
    if (la.a[i].i32 != 0 && la.a[i].i32 != 1)
      return fail(MTL_ERR_ARGUMENT, "quantize_fp8: argument %d must be 0 or 1, got %d", i + 1, la.a[i].i32);
  const bool gather = la.a[5].kind == MTL_ARG_PTR;
  if (gather && batch > 1) return fail(MTL_ERR_UNSUPPORTED, "quantize_fp8: rows_of goes with a batch of one, got %lld", (long long)batch);
  if (!gather && xrows != R)
    return fail(MTL_ERR_ARGUMENT, "quantize_fp8: without rows_of the input has as many rows as the output: %lld, got %lld", (long long)R,
                (long long)xrows);
  const bool q = la.a[0].ptr, s = la.a[1].ptr, qt = la.a[2].ptr, st = la.a[3].ptr, none = batch == 0 || R == 0 || C == 0;
  if (!none && (q != s || qt != st || (!q && !qt)))
    return fail(MTL_ERR_ARGUMENT, "quantize_fp8: give the codes and the scales of the row form, of the transposed form, or of both");
  const int64_t rb = (R + 127) / 128, cb = (C + 127) / 128, per = la.a[10].i32 ? 2 : 4;
  const bool square = block == 128;
  const uint64_t need[6] = {bytes_of({batch, R, up(C, 16)}), bytes_of({batch, cb, square ? rb : R, 4}), bytes_of({batch, C, up(R, 16)}),
                            bytes_of({batch, rb, square ? cb : C, 4}), bytes_of({gather ? 1 : batch, xrows, C, per}), bytes_of({R, 4})};
  const char* what[6] = {"the codes", "the scales", "the transposed codes", "the transposed scales", "the input", "rows_of"};
  const unsigned align[6] = {15, 3, 15, 3, la.a[10].i32 ? 1u : 3u, 3};
  for (int i = 0; i < 6; ++i) {
    if (la.a[i].kind == MTL_ARG_PTR && !la.a[i].ptr && need[i])  // given, but without an address: not the same as left out
      return fail(MTL_ERR_ARGUMENT, "quantize_fp8: %s must be a device buffer", what[i]);
    if (!la.a[i].ptr) continue;
    if (bytes[i] && bytes[i] < need[i])
      return fail(MTL_ERR_ARGUMENT, "quantize_fp8: %s: %llu bytes, the launch touches %llu", what[i], (unsigned long long)bytes[i],
                  (unsigned long long)need[i]);
    if (la.a[i].ptr & align[i])
      return fail(MTL_ERR_ARGUMENT, "quantize_fp8: %s must be %u-byte aligned", what[i], align[i] + 1);
  }
  if (bytes_of({batch, std::max<int64_t>(1, (R + 15) / 16), std::max<int64_t>(1, cb)}) > INT_MAX)
    return fail(MTL_ERR_UNSUPPORTED, "quantize_fp8: more than 2^31 tiles");
  return MTL_OK;
}

template <typename T, bool E5M2>
static void quantize_launch(const QuantArgs& a, int64_t batch, int block, int sms, cudaStream_t st) {
  if (block == 1 && !a.qt) {
    // four blocks of a row a thread group once that leaves every SM several CTAs
    const unsigned row_tiles = (unsigned)((a.R + 15) / 16);
    const bool four = batch * row_tiles * a.cb >= 8 * (int64_t)sms;
    const unsigned col_tiles = (unsigned)(four ? (a.cb + 3) / 4 : a.cb), grid = (unsigned)batch * row_tiles * col_tiles;
    if (four)
      quantize_rows_kernel<T, 4, E5M2><<<grid, kQuantThreads, 0, st>>>(a, row_tiles, col_tiles);
    else
      quantize_rows_kernel<T, 1, E5M2><<<grid, kQuantThreads, 0, st>>>(a, row_tiles, col_tiles);
  } else {
    quantize_tile_kernel<T, E5M2><<<(unsigned)(batch * a.rb * a.cb), kQuantThreads, 0, st>>>(a, block == 128);
  }
}

mtl_status quantize_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  QuantArgs a = {};
  a.q = reinterpret_cast<uint8_t*>(la.a[0].ptr);
  a.s = reinterpret_cast<float*>(la.a[1].ptr);
  a.qt = reinterpret_cast<uint8_t*>(la.a[2].ptr);
  a.st = reinterpret_cast<float*>(la.a[3].ptr);
  a.x = reinterpret_cast<const void*>(la.a[4].ptr);
  a.rows_of = reinterpret_cast<const int*>(la.a[5].ptr);
  a.R = la.a[6].i32;
  a.C = la.a[7].i32;
  a.xrows = la.a[8].i32;
  a.Cp = up(a.C, 16);
  a.Rp = up(a.R, 16);
  a.rb = (a.R + 127) / 128;
  a.cb = (a.C + 127) / 128;
  const int block = la.a[9].i32, bf16 = la.a[10].i32;
  a.pow2 = la.a[12].i32;
  a.vec = la.a[4].ptr % 16 == 0 && a.C % (bf16 ? 8 : 4) == 0;
  const int64_t batch = la.nd[0];
  cudaStream_t st = (cudaStream_t)stream;
  if (batch == 0 || a.R == 0 || a.C == 0) return MTL_OK;
  const bool e5m2 = la.a[11].i32;
  if (bf16)
    e5m2 ? quantize_launch<uint16_t, true>(a, batch, block, la.sm_count, st) : quantize_launch<uint16_t, false>(a, batch, block, la.sm_count, st);
  else
    e5m2 ? quantize_launch<float, true>(a, batch, block, la.sm_count, st) : quantize_launch<float, false>(a, batch, block, la.sm_count, st);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "quantize_fp8: %s", cudaGetErrorString(e));
}

}  // namespace mtl
