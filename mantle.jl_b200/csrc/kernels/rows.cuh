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

// How B threads share a row, eight values each at a time: with VEC thread t holds columns
// (u B + t) 8 .. + 8, which needs rows that start on 16 bytes and C a multiple of 8;
// without it columns (8 u + i) B + t, so that a warp's access is one run of neighbouring
// values wherever the row starts. Columns from C on are zeros and are not stored. (For rows
// of odd length the 16-byte words around them, shifted into place, took more: rms_norm with a
// residual on 8192 x 4095 bfloat16 117 us where this took 77, 5001 x 4013 float 48 and 33.)
template <int B, bool VEC, typename T>
__device__ __forceinline__ void load_part(float (&v)[8], const T* row, int C, int tid, int u) {
  if constexpr (VEC) {
    const int c = (u * B + tid) * 8;
    if (c < C) {
      load8(v, row + c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (u * 8 + i) * B + tid;
      v[i] = c < C ? to_f32(row[c]) : 0.0f;
    }
  }
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

// ── chunks: the neighbouring columns of 16 bytes, as pairs ──────────────────
// A row that starts off 16 bytes is cut where the 16 bytes are: its first chunk begins
// up to seven columns before the row, its last ends behind it. What lies outside the row
// is read (but not outside the tensor), taken for zeros, and not written. Rows a
// multiple of eight apart are cut alike.
template <typename T>
constexpr int kWide = 16 / (int)sizeof(T);  // values of a chunk
template <typename T>
constexpr int kPairs = kWide<T> / 2;
struct Chunk {
  int c;      // its first column
  bool on;    // it has a column of the row
  bool edge;  // and one outside
};
template <typename T>
__device__ __forceinline__ Chunk chunk_of(int j, int phase, int C) {
  Chunk k;
  k.c = j * kWide<T> - phase;
  k.on = k.c < C;
  k.edge = k.c < 0 || k.c + kWide<T> > C;
  return k;
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  float2 o;
  asm("{ .reg .b64 a, b, c; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 a, a, b, c; mov.b64 {%0, %1}, a; }"
      : "=f"(o.x), "=f"(o.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
  return o;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <int P>
__device__ __forceinline__ void only_inside(float2 (&v)[P], const Chunk& k, int C) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = k.c + 2 * i;
    if (c < 0 || c >= C) v[i].x = 0.0f;
    if (c + 1 < 0 || c + 1 >= C) v[i].y = 0.0f;
  }
}
// One value after the other, whatever the address and its type.
template <int P, typename T>
__device__ __forceinline__ void load_each(float2 (&v)[P], const T* row, const Chunk& k, int C) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = k.c + 2 * i;
    v[i].x = c >= 0 && c < C ? to_f32(row[c]) : 0.0f;
    v[i].y = c + 1 >= 0 && c + 1 < C ? to_f32(row[c + 1]) : 0.0f;
  }
}
template <int P, typename T>
__device__ __forceinline__ void store_each(T* row, const float2 (&v)[P], const Chunk& k, int C) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = k.c + 2 * i;
    if (c >= 0 && c < C) row[c] = from_f32<T>(v[i].x);
    if (c + 1 >= 0 && c + 1 < C) row[c + 1] = from_f32<T>(v[i].y);
  }
}
__device__ __forceinline__ void load_pairs(float2 (&v)[2], const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w);
}
__device__ __forceinline__ void load_pairs(float2 (&v)[4], const uint16_t* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  v[0] = make_float2(bf16_lo(u.x), bf16_hi(u.x)), v[1] = make_float2(bf16_lo(u.y), bf16_hi(u.y));
  v[2] = make_float2(bf16_lo(u.z), bf16_hi(u.z)), v[3] = make_float2(bf16_lo(u.w), bf16_hi(u.w));
}
__device__ __forceinline__ void store_pairs(float* p, const float2 (&v)[2]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
}
__device__ __forceinline__ void store_pairs(uint16_t* p, const float2 (&v)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0].x, v[0].y), bf16_pair(v[1].x, v[1].y), bf16_pair(v[2].x, v[2].y), bf16_pair(v[3].x, v[3].y));
}
// A chunk of row `row` of a tensor of `total` values. `vec`: chunks start on 16 bytes.
template <bool PHASED, typename T>
__device__ __forceinline__ void load_chunk(float2 (&v)[kPairs<T>], const T* x, int64_t row, const Chunk& k, int C, int64_t total, bool vec) {
  const int64_t at = row * C + k.c;
  if (!k.on) {
#pragma unroll
    for (int i = 0; i < kPairs<T>; ++i) v[i] = make_float2(0.0f, 0.0f);
  } else if (!PHASED || (vec && at >= 0 && at + kWide<T> <= total)) {
    load_pairs(v, x + at);
    if (PHASED && k.edge) only_inside(v, k, C);
  } else {
    load_each(v, x + row * C, k, C);
  }
}
template <bool PHASED, typename T>
__device__ __forceinline__ void store_chunk(T* x, int64_t row, const float2 (&v)[kPairs<T>], const Chunk& k, int C, bool vec) {
  if (!PHASED || (vec && !k.edge)) {
    if (k.on) store_pairs(x + row * C + k.c, v);
  } else if (k.on) {
    store_each(x + row * C, v, k, C);
  }
}
// The same by way of shared memory: chunk j of a row's image, which its thread alone
// writes and reads, 16 bytes at 16 j. (What lies outside the row comes as it is.)
template <bool PHASED, typename T>
__device__ __forceinline__ void copy_chunk(uint8_t* image, int j, const T* x, int64_t row, const Chunk& k, int C, int64_t total) {
  if (!k.on) return;
  const int64_t at = row * C + k.c;
  if (!PHASED || (at >= 0 && at + kWide<T> <= total)) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(image + j * 16)), "l"(x + at) : "memory");
  } else {
    for (int i = 0; i < kWide<T>; ++i) {
      const int c = k.c + i;
      reinterpret_cast<T*>(image + j * 16)[i] = c >= 0 && c < C ? x[row * C + c] : T(0);
    }
  }
}
template <typename T>
__device__ __forceinline__ void chunk_in(float2 (&v)[kPairs<T>], const uint8_t* image, int j) {
  load_pairs(v, reinterpret_cast<const T*>(image + j * 16));
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// At most `pending` (0 .. 6) of this thread's latest groups are still on their way.
__device__ __forceinline__ void copies_wait(int pending) {
  switch (pending) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
  }
}
// Dynamic shared memory above 48 KiB, allowed a kernel once on each device.
template <typename F>
inline cudaError_t allow_shared(F* kernel, int bytes, int device, unsigned long long* done) {
  if (device >= 0 && device < 64 && (__atomic_load_n(done, __ATOMIC_RELAXED) >> device & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device >= 0 && device < 64) __atomic_fetch_or(done, 1ull << device, __ATOMIC_RELAXED);
  return e;
}
// How far behind a 16-byte boundary an address lies, in values.
inline int phase_of(uint64_t ptr, int size) { return (int)(ptr % 16 / size); }

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
