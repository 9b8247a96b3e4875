// What the kernels that write 8-bit codes share: a block's scale from its largest
// magnitude, the conversion to codes, and the maxima of a row's blocks. The
// definitions are at the top of quantize.cu.
#pragma once

#include <cstdint>

namespace mtl {

__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }

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

}  // namespace mtl
