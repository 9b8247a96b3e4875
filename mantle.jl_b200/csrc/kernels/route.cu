// Routing of tokens to experts: scores, the choice of experts, their weights and the rows'
// order by expert, which quantize_fp8's rows_of and the grouped products' offsets take; and
// the logits' gradient.
//
// With the logits l of a token:
//
//   score    s = softmax(l) or sigmoid(l); an expert whose logit is -inf is masked
//   key      s + bias, or where there is no bias the order of l itself
//   groups   the E experts lie in `groups` runs; a group's value is the sum of its `best`
//            largest keys, and only the `top_groups` groups of the largest values stay
//   ids      the `top` largest keys in falling order
//   weight   scale * s, or scale * s / (sum of the chosen s)
//
// Ties go to the lower index. The bias moves the choice alone. Where fewer experts can be
// chosen than asked for, and for a token that is not live, an id is -1 and its weight 0. A
// NaN among a token's logits (or the biases, or +inf under softmax) makes its ids -1 and
// its weights NaN.
//
// Keys are compared as their 64-bit values are: a score rounded to 32 bits would tie
// experts, or turn their order round, wherever two keys are within 1e-7. Weights are
// 32-bit. Over their sum they are computed from the chosen logits alone (for softmax the
// sum over all experts cancels), relative to the largest, so that no sum is ever zero.
//
// The order of rows: slot s = token * top + j. Rows are the slots with an expert, by
// expert, then slot; rows_of[row] is the slot's token (-1 behind the last row),
// row_at[s] its row (-1 without an expert), offsets[e] the first row of expert e.
//
// The gradient, with g the weights' gradient, c = scale, S the chosen and sums over S:
//   softmax              c p_e ([e in S] g_e - sum g p)   over all experts
//   softmax, over sum    c u_e (g_e - sum g u)            u = p / sum p, on S
//   sigmoid              c s_e (1 - s_e) g_e              on S
//   sigmoid, over sum    c u_e (1 - s_e) (g_e - sum g u)  u = s / sum s, on S

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "../mtl_internal.hpp"
#include "rows.cuh"

namespace mtl {

constexpr int kMaxExperts = 1024;  // as the grouped products
constexpr int kMaxTop = 32;        // a lane each

struct RouteArgs {
  int* ids;
  float* weights;
  const void* logits;
  const float* bias;
  const int* live;
  int64_t T;
  int E, top, groups, top_groups, best;
  int sigmoid, renorm;
  float scale;
};

// 64-bit keys as integers of the same order.
__device__ __forceinline__ unsigned long long ordered(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);  // -0 as 0
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
constexpr unsigned long long kNoKey = 0x000fffffffffffffull;  // ordered(-infinity)

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, d);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// The weights of a token's chosen experts: lane j has slot j's logit, or -inf for none.
__device__ __forceinline__ float weight_of(float l, bool valid, float most, float total, int sigmoid, int renorm, float scale) {
  float s;
  if (!renorm) {
    s = sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - most) / total;
  } else if (sigmoid) {
    // s_i up to a common factor: e^min(l, 0) / (1 + e^-|l|)
    const float m = fminf(warp_max(valid ? l : -INFINITY), 0.0f);
    s = valid ? expf(fminf(l, 0.0f) - m) / (1.0f + expf(-fabsf(l))) : 0.0f;
    s = s / warp_sum(s);
  } else {
    const float m = warp_max(valid ? l : -INFINITY);
    s = valid ? expf(l - m) : 0.0f;
    s = s / warp_sum(s);
  }
  return valid ? s * scale : 0.0f;
}

// A warp a token; lane i holds experts i, i + 32, ...: P of them.
template <typename T, int P>
__global__ void __launch_bounds__(128) route_kernel(RouteArgs a) {
  extern __shared__ unsigned long long group_keys[];  // a warp's groups x 2
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * 4 + warp;
  if (t >= a.T) return;
  const int E = a.E;
  const T* logits = static_cast<const T*>(a.logits) + t * E;
  float l[P];
  bool bad = false;
  float most = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int e = p * 32 + lane;
    l[p] = e < E ? to_f32(logits[e]) : -INFINITY;
    bad |= isnan(l[p]) || (a.bias && e < E && isnan(a.bias[e]));
    most = fmaxf(most, l[p]);
  }
  most = warp_max(most);
  bad = __any_sync(0xffffffffu, bad || (!a.sigmoid && most == INFINITY));
  const bool none = most == -INFINITY || (a.live && !a.live[t]);
  if (bad || none) {
    if (lane < a.top) {
      a.ids[t * a.top + lane] = -1;
      a.weights[t * a.top + lane] = none && a.live && !a.live[t] ? 0.0f : bad ? NAN : 0.0f;
    }
    return;
  }
  float total = 0.0f;
  if (!a.sigmoid) {
#pragma unroll
    for (int p = 0; p < P; ++p) total += expf(l[p] - most);
    total = warp_sum(total);
  }
  unsigned long long key[P];
  if (a.bias) {
    double s[P], all = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      s[p] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)l[p])) : exp((double)l[p] - (double)most);
      all += s[p];
    }
    if (!a.sigmoid) {
      all = warp_sum(all);
#pragma unroll
      for (int p = 0; p < P; ++p) s[p] /= all;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int e = p * 32 + lane;
      key[p] = e < E && l[p] != -INFINITY ? ordered(s[p] + (double)a.bias[e]) : kNoKey;
    }
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) key[p] = ordered((double)l[p]);
  }
  if (a.groups > 1) {
    // each group's best keys, one group after the other
    const int per = E / a.groups;
    unsigned long long* value = group_keys + warp * a.groups;
    for (int g = 0; g < a.groups; ++g) {
      const int lo = g * per, hi = lo + per;
      unsigned long long first = kNoKey, second = kNoKey;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int e = p * 32 + lane;
        const unsigned long long k = e >= lo && e < hi ? key[p] : kNoKey;
        second = max(second, min(first, k));
        first = max(first, k);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const unsigned long long f = __shfl_xor_sync(0xffffffffu, first, d), s = __shfl_xor_sync(0xffffffffu, second, d);
        second = max(max(second, s), min(first, f));
        first = max(first, f);
      }
      if (a.best > 1 && first != kNoKey) {
        // without a bias the keys are logits: their scores, up to softmax's common factor
        const auto score = [&](unsigned long long k) {
          const double v = __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
          return a.bias ? v : a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)most);
        };
        first = ordered(score(first) + (second != kNoKey ? score(second) : 0.0));
      }
      if (lane == 0) value[g] = first;
    }
    __syncwarp();
    // a group stays if fewer than top_groups are ahead of it
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int e = p * 32 + lane;
      if (e < E) {
        const int g = e / per;
        int ahead = 0;
        for (int o = 0; o < a.groups; ++o) ahead += value[o] > value[g] || (value[o] == value[g] && o < g);
        if (ahead >= a.top_groups) key[p] = kNoKey;
      }
    }
  }
  // one choice after the other: the largest key, its lowest index
  int id = -1;
  for (int j = 0; j < a.top; ++j) {
    unsigned long long k = kNoKey;
#pragma unroll
    for (int p = 0; p < P; ++p) k = max(k, key[p]);
    k = warp_max(k);
    if (k == kNoKey) break;
    int e = INT_MAX;
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
      if (key[p] == k) e = p * 32 + lane;
    e = __reduce_min_sync(0xffffffffu, e);
    if (lane == j) id = e;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (e == p * 32 + lane) key[p] = kNoKey;
  }
  const float chosen = id >= 0 ? to_f32(logits[id]) : -INFINITY;
  const float w = weight_of(chosen, id >= 0, most, total, a.sigmoid, a.renorm, a.scale);
  if (lane < a.top) {
    a.ids[t * a.top + lane] = id;
    a.weights[t * a.top + lane] = w;
  }
}

// ── the rows' order ─────────────────────────────────────────────────────────
// A counting sort by one cluster. Each warp has a run of slots and a counter for each
// expert; the counters' prefix sums over warps, then over CTAs (whose totals the others
// read in their shared memory), then over experts give each warp where its rows of each
// expert start. So the order is that of the slots whatever the warps' timing.
constexpr int kOrderWarps = 32;
struct OrderArgs {
  const int* ids;
  int* offsets;
  int* rows_of;
  int* row_at;
  int64_t n;
  int E, top;
};

__global__ void __launch_bounds__(kOrderWarps * 32) order_rows_kernel(OrderArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ int order_smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int E = a.E, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  int* count = order_smem;                // [warp][expert]
  int* total = count + kOrderWarps * E;   // this CTA's rows of each expert
  int* start = total + E;                 // the first row of each expert that is this CTA's
  int* sums = start + E;                  // [32] of the scan, and the number of rows
  for (int i = threadIdx.x; i < kOrderWarps * E; i += blockDim.x) count[i] = 0;
  const int64_t steps = (a.n + 31) / 32, per = (steps + (int64_t)ctas * kOrderWarps - 1) / ((int64_t)ctas * kOrderWarps) * 32;
  const int64_t lo = min(a.n, ((int64_t)rank * kOrderWarps + warp) * per), hi = min(a.n, lo + per);
  __syncthreads();
  int* mine = count + warp * E;
  for (int64_t s = lo + lane; s < hi; s += 32) {
    const int id = a.ids[s];
    if ((unsigned)id < (unsigned)E) atomicAdd(mine + id, 1);
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < E) {
    int run = 0;
    for (int w = 0; w < kOrderWarps; ++w) {
      const int c = count[w * E + e];
      count[w * E + e] = run;
      run += c;
    }
    total[e] = run;
  }
  cluster.sync();
  int before = 0, all = 0;
  if (e < E)
    for (int r = 0; r < ctas; ++r) {
      const int c = cluster.map_shared_rank(total, r)[e];
      if (r < rank) before += c;
      all += c;
    }
  int scan = all;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += o;
  }
  if (lane == 31) sums[warp] = scan;
  __syncthreads();
  if (warp == 0) {
    int v = sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    sums[lane] = v;
  }
  __syncthreads();
  const int first = scan - all + (warp ? sums[warp - 1] : 0), rows = sums[31];
  if (e < E) {
    start[e] = first + before;
    if (rank == 0) {
      a.offsets[e] = first;
      if (e == E - 1) a.offsets[E] = rows;
    }
  }
  cluster.sync();  // nobody leaves while its totals are read
  for (int64_t s = lo + lane; s - lane < hi; s += 32) {
    const int id = s < hi ? a.ids[s] : -1;
    const bool valid = (unsigned)id < (unsigned)E;
    const unsigned peers = __match_any_sync(0xffffffffu, valid ? id : -1);
    if (valid) {
      const int at = start[id] + mine[id] + __popc(peers & ((1u << lane) - 1));
      a.rows_of[at] = (int)((uint32_t)s / (uint32_t)a.top);
      a.row_at[s] = at;
    } else if (s < hi) {
      a.row_at[s] = -1;
    }
    __syncwarp();
    if (valid && (peers & ((1u << lane) - 1)) == 0) mine[id] += __popc(peers);
    __syncwarp();
  }
  for (int64_t r = rows + (int64_t)rank * blockDim.x + threadIdx.x; r < a.n; r += (int64_t)ctas * blockDim.x) a.rows_of[r] = -1;
}

// ── the gradient ────────────────────────────────────────────────────────────
struct RouteGradArgs {
  void* dlogits;
  const float* dweights;
  const void* logits;
  const int* ids;
  int64_t T;
  int E, top, sigmoid, renorm;
  float scale;
};

template <typename T, int P>
__global__ void __launch_bounds__(128) route_grad_kernel(RouteGradArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= a.T) return;
  const int E = a.E;
  const T* logits = static_cast<const T*>(a.logits) + t * E;
  T* out = static_cast<T*>(a.dlogits) + t * E;
  int id = lane < a.top ? a.ids[t * a.top + lane] : -1;
  if ((unsigned)id >= (unsigned)E) id = -1;
  const bool valid = id >= 0;
  float g = valid ? a.dweights[t * a.top + lane] : 0.0f;
  const float l = valid ? to_f32(logits[id]) : -INFINITY;
  float p[P], most = -INFINITY, total = 1.0f;
  const bool dense = !a.sigmoid && !a.renorm;
  if (dense) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int e = i * 32 + lane;
      p[i] = e < E ? to_f32(logits[e]) : -INFINITY;
      most = fmaxf(most, p[i]);
    }
    most = warp_max(most);
    if (most == -INFINITY) most = 0.0f;  // every expert masked: all of p is 0
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) total += p[i] = expf(p[i] - most);
    total = warp_sum(total);
    if (total == 0.0f) total = 1.0f;
  }
  const float u = weight_of(l, valid, most, total, a.sigmoid, a.renorm, 1.0f);
  const float mean = a.sigmoid && !a.renorm ? 0.0f : warp_sum(g * u);
  float d;
  if (dense) {
    // an expert named twice: its slots' gradients together
    const unsigned peers = __match_any_sync(0xffffffffu, valid ? id : -1 - lane);
    if (__any_sync(0xffffffffu, peers & (peers - 1))) {
      float sum = 0.0f;
      for (int j = 0; j < 32; ++j) {
        const float o = __shfl_sync(0xffffffffu, g, j);
        if (peers >> j & 1) sum += o;
      }
      g = sum;
    }
    d = u * (g - mean);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int e = i * 32 + lane;
      if (e < E) out[e] = from_f32<T>(-a.scale * (p[i] / total) * mean);
    }
  } else {
    d = u * (g - mean);
    if (a.sigmoid) d *= 1.0f / (1.0f + expf(l));  // 1 - s
    const unsigned peers = __match_any_sync(0xffffffffu, valid ? id : -1 - lane);
    if (__any_sync(0xffffffffu, peers & (peers - 1))) {
      float sum = 0.0f;
      for (int j = 0; j < 32; ++j) {
        const float o = __shfl_sync(0xffffffffu, d, j);
        if (peers >> j & 1) sum += o;
      }
      d = sum;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int e = i * 32 + lane;
      if (e < E) out[e] = from_f32<T>(0.0f);
    }
  }
  __syncwarp();
  if (valid) out[id] = from_f32<T>(a.scale * d);
}

// ── host side ───────────────────────────────────────────────────────────────
static mtl_status route_sizes(const char* kernel, const LaunchArgs& la, int E, int top, float scale) {
  if (la.ndim != 1) return fail(MTL_ERR_ARGUMENT, "%s: ndrange must be one-dimensional (the tokens)", kernel);
  if (la.nd[0] < 0 || E < 1) return fail(MTL_ERR_ARGUMENT, "%s: negative dimension, or no experts", kernel);
  if (E > kMaxExperts) return fail(MTL_ERR_UNSUPPORTED, "%s: more than %d experts: %d", kernel, kMaxExperts, E);
  if (top < 1 || top > E || top > kMaxTop)
    return fail(MTL_ERR_ARGUMENT, "%s: top must be 1 .. %d and no more than the experts, got %d of %d", kernel, kMaxTop, top, E);
  if (bytes_of({la.nd[0], top}) > INT_MAX) return fail(MTL_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots", kernel);
  if (!std::isfinite(scale)) return fail(MTL_ERR_ARGUMENT, "%s: scale must be finite, got %g", kernel, scale);
  return MTL_OK;
}

// Arguments: ids (B), weights (B), offsets (b), rows_of (b), row_at (b), logits (B), bias
// (b), live (b), E, top, groups, top_groups, best, score (0 softmax, 1 sigmoid), renorm,
// type of the logits (0 f32, 1 bf16) (i), scale (f); ndrange = tokens.
mtl_status route_experts_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int64_t T = la.nd[0];
  const int E = la.a[8].i32, top = la.a[9].i32, groups = la.a[10].i32, top_groups = la.a[11].i32, best = la.a[12].i32;
  if (mtl_status s = route_sizes("route_experts", la, E, top, la.a[16].f32)) return s;
  if (mtl_status s = check_flags("route_experts", la, {13, 14, 15})) return s;
  if (groups < 1 || groups > E || E % groups)
    return fail(MTL_ERR_ARGUMENT, "route_experts: groups must divide the experts: %d of %d", groups, E);
  if (top_groups < 1 || top_groups > groups)
    return fail(MTL_ERR_ARGUMENT, "route_experts: top_groups must be 1 .. groups, got %d of %d", top_groups, groups);
  if (best < 1 || best > 2 || best > E / groups)
    return fail(MTL_ERR_ARGUMENT, "route_experts: a group's value is its best key or the sum of its best two, got %d of %d", best, E / groups);
  if (given(la, 2) != given(la, 3) || given(la, 2) != given(la, 4))
    return fail(MTL_ERR_ARGUMENT, "route_experts: offsets, rows_of and row_at go together");
  const uint64_t slots = bytes_of({T, top, 4}), per = la.a[15].i32 ? 2 : 4;
  return check_operands("route_experts", la, bytes,
                        {{"ids", slots, 4},
                         {"the weights", slots, 4},
                         {"offsets", bytes_of({E + 1, 4}), 4},
                         {"rows_of", slots, 4},
                         {"row_at", slots, 4},
                         {"the logits", bytes_of({T, E, (int64_t)per}), (unsigned)per},
                         {"the bias", T ? bytes_of({E, 4}) : 0, 4},
                         {"live", bytes_of({T, 4}), 4}});
}

template <typename T>
static void route_launch(const RouteArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.T + 3) / 4);
  const size_t smem = a.groups > 1 ? 4 * sizeof(unsigned long long) * a.groups : 0;
  if (a.E <= 32)
    route_kernel<T, 1><<<grid, 128, smem, st>>>(a);
  else if (a.E <= 64)
    route_kernel<T, 2><<<grid, 128, smem, st>>>(a);
  else if (a.E <= 128)
    route_kernel<T, 4><<<grid, 128, smem, st>>>(a);
  else if (a.E <= 256)
    route_kernel<T, 8><<<grid, 128, smem, st>>>(a);
  else if (a.E <= 512)
    route_kernel<T, 16><<<grid, 128, smem, st>>>(a);
  else
    route_kernel<T, 32><<<grid, 128, smem, st>>>(a);
}

mtl_status route_experts_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  RouteArgs a = {};
  a.ids = reinterpret_cast<int*>(la.a[0].ptr);
  a.weights = reinterpret_cast<float*>(la.a[1].ptr);
  a.logits = reinterpret_cast<const void*>(la.a[5].ptr);
  a.bias = reinterpret_cast<const float*>(la.a[6].ptr);
  a.live = reinterpret_cast<const int*>(la.a[7].ptr);
  a.T = la.nd[0];
  a.E = la.a[8].i32;
  a.top = la.a[9].i32;
  a.groups = la.a[10].i32;
  a.top_groups = la.a[11].i32;
  a.best = la.a[12].i32;
  a.sigmoid = la.a[13].i32;
  a.renorm = la.a[14].i32;
  a.scale = la.a[16].f32;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.T) la.a[15].i32 ? route_launch<uint16_t>(a, st) : route_launch<float>(a, st);
  if (given(la, 2)) {
    OrderArgs o = {};
    o.ids = a.ids;
    o.offsets = reinterpret_cast<int*>(la.a[2].ptr);
    o.rows_of = reinterpret_cast<int*>(la.a[3].ptr);
    o.row_at = reinterpret_cast<int*>(la.a[4].ptr);
    o.n = a.T * a.top;
    o.E = a.E;
    o.top = a.top;
    const size_t smem = sizeof(int) * ((kOrderWarps + 2) * (size_t)a.E + 32);
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(order_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return fail(MTL_ERR_CUDA, "route_experts: %s", cudaGetErrorString(e));
    }
    order_rows_kernel<<<1, kOrderWarps * 32, smem, st>>>(o);
  }
  return launched("route_experts");
}

// Arguments: dlogits (B), dweights (B), logits (B), ids (B), E, top, score, renorm, type of
// the logits and dlogits (i), scale (f); ndrange = tokens.
mtl_status route_experts_grad_check(const LaunchArgs& la, const uint64_t* bytes) {
  const int64_t T = la.nd[0];
  const int E = la.a[4].i32, top = la.a[5].i32;
  if (mtl_status s = route_sizes("route_experts_grad", la, E, top, la.a[9].f32)) return s;
  if (mtl_status s = check_flags("route_experts_grad", la, {6, 7, 8})) return s;
  const int64_t per = la.a[8].i32 ? 2 : 4;
  const uint64_t all = bytes_of({T, E, per}), slots = bytes_of({T, top, 4});
  return check_operands("route_experts_grad", la, bytes,
                        {{"dlogits", all, (unsigned)per}, {"the weights' gradient", slots, 4}, {"the logits", all, (unsigned)per}, {"ids", slots, 4}});
}

template <typename T>
static void route_grad_launch(const RouteGradArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.T + 3) / 4);
  if (a.E <= 32)
    route_grad_kernel<T, 1><<<grid, 128, 0, st>>>(a);
  else if (a.E <= 64)
    route_grad_kernel<T, 2><<<grid, 128, 0, st>>>(a);
  else if (a.E <= 128)
    route_grad_kernel<T, 4><<<grid, 128, 0, st>>>(a);
  else if (a.E <= 256)
    route_grad_kernel<T, 8><<<grid, 128, 0, st>>>(a);
  else if (a.E <= 512)
    route_grad_kernel<T, 16><<<grid, 128, 0, st>>>(a);
  else
    route_grad_kernel<T, 32><<<grid, 128, 0, st>>>(a);
}

mtl_status route_experts_grad_run(const LaunchArgs& la, void*, uint64_t, void* stream) {
  RouteGradArgs a = {};
  a.dlogits = reinterpret_cast<void*>(la.a[0].ptr);
  a.dweights = reinterpret_cast<const float*>(la.a[1].ptr);
  a.logits = reinterpret_cast<const void*>(la.a[2].ptr);
  a.ids = reinterpret_cast<const int*>(la.a[3].ptr);
  a.T = la.nd[0];
  a.E = la.a[4].i32;
  a.top = la.a[5].i32;
  a.sigmoid = la.a[6].i32;
  a.renorm = la.a[7].i32;
  a.scale = la.a[9].f32;
  if (a.T == 0) return MTL_OK;
  la.a[8].i32 ? route_grad_launch<uint16_t>(a, (cudaStream_t)stream) : route_grad_launch<float>(a, (cudaStream_t)stream);
  return launched("route_experts_grad");
}

}  // namespace mtl
