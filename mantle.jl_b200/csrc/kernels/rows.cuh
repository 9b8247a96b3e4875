// What the kernels over rows of values share: eight values of either element type
// at a time, sums over a row's threads, and the host's checks of operands.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "../mtl_internal.hpp"
#include "fp8_codes.cuh"

namespace mtl {

// ── values: float, or bfloat16 as its bits ──────────────────────────────────
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float v) {  // to the nearest, ties to even
  return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t u;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  return u;
}

// Eight neighbouring values from or to an address of 16 bytes' alignment.
__device__ __forceinline__ void load8(float (&v)[8], const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(float (&v)[8], const uint16_t* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
  v[4] = bf16_lo(u.z), v[5] = bf16_hi(u.z), v[6] = bf16_lo(u.w), v[7] = bf16_hi(u.w);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
}

// How B threads share a row: with VEC thread t holds columns (u B + t) 8 .. + 8, which
// needs rows that start on 16 bytes and C a multiple of 8; without it columns
// (8 u + i) B + t, so that a warp's access is one run of neighbouring values wherever
// the row starts. Columns from C on are zeros and are not stored.
template <int B, int N, bool VEC, typename T>
__device__ __forceinline__ void load_row(float (&v)[N][8], const T* row, int C, int tid) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if constexpr (VEC) {
      const int c = (u * B + tid) * 8;
      if (c < C) {
        load8(v[u], row + c);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = (u * 8 + i) * B + tid;
        v[u][i] = c < C ? to_f32(row[c]) : 0.0f;
      }
    }
  }
}
template <int B, bool VEC, typename T>
__device__ __forceinline__ void load_part(float (&v)[8], const T* row, int C, int tid, int u) {
  float one[1][8];
  if constexpr (VEC)
    load_row<B, 1, true>(one, row, C, u * B + tid);
  else
    load_row<B, 1, false>(one, row, C, u * 8 * B + tid);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = one[0][i];
}
template <int B, bool VEC, typename T>
__device__ __forceinline__ void store_part(T* row, const float (&v)[8], int C, int tid, int u) {
  if constexpr (VEC) {
    const int c = (u * B + tid) * 8;
    if (c < C) store8(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (u * 8 + i) * B + tid;
      if (c < C) row[c] = from_f32<T>(v[i]);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// ── host: the buffers of a launch ───────────────────────────────────────────
struct Operand {
  const char* what;
  uint64_t need;   // bytes the launch touches
  unsigned align;  // in bytes
};
// Argument i of the launch is the i-th operand. One left out is the caller's to allow.
inline mtl_status check_operands(const char* kernel, const LaunchArgs& la, const uint64_t* bytes, std::initializer_list<Operand> ops) {
  int i = 0;
  for (const Operand& o : ops) {
    const Arg& x = la.a[i];
    if (x.kind == MTL_ARG_PTR && !x.ptr && o.need)  // given, but without an address: not the same as left out
      return fail(MTL_ERR_ARGUMENT, "%s: %s must be a device buffer", kernel, o.what);
    if (x.ptr) {
      if (bytes[i] && bytes[i] < o.need)
        return fail(MTL_ERR_ARGUMENT, "%s: %s: %llu bytes, the launch touches %llu", kernel, o.what, (unsigned long long)bytes[i],
                    (unsigned long long)o.need);
      if (x.ptr % o.align) return fail(MTL_ERR_ARGUMENT, "%s: %s must be %u-byte aligned", kernel, o.what, o.align);
    }
    ++i;
  }
  return MTL_OK;
}
// Scalars that are 0 or 1.
inline mtl_status check_flags(const char* kernel, const LaunchArgs& la, std::initializer_list<int> args) {
  for (int i : args)
    if (la.a[i].i32 != 0 && la.a[i].i32 != 1)
      return fail(MTL_ERR_ARGUMENT, "%s: argument %d must be 0 or 1, got %d", kernel, i + 1, la.a[i].i32);
  return MTL_OK;
}
inline bool given(const LaunchArgs& la, int i) { return la.a[i].kind == MTL_ARG_PTR; }
inline mtl_status launched(const char* kernel) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MTL_OK : fail(MTL_ERR_CUDA, "%s: %s", kernel, cudaGetErrorString(e));
}

}  // namespace mtl
