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
//   softmax              c p_e ([e in S] g_e - sum g p)   over all experts (0 where S is empty)
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
#include "tc_common.cuh"

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
  int cut, lanes, each;  // route_token: the runs that lie on lanes, the lanes of one, the experts of a lane
};

// Keys as integers of the same order, -0 as 0.
template <typename K>
struct Key;
template <>
struct Key<uint32_t> {
  static constexpr uint32_t kNone = 0x007fffffu;  // -infinity's
  static __device__ __forceinline__ uint32_t of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }
  static __device__ __forceinline__ uint32_t most(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
};
template <>
struct Key<unsigned long long> {
  static constexpr unsigned long long kNone = 0x000fffffffffffffull;
  static __device__ __forceinline__ unsigned long long of(double v) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
  }
  static __device__ __forceinline__ double value(unsigned long long k) {
    return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
  }
  // of the warp's, the upper halves first
  static __device__ __forceinline__ unsigned long long most(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (unsigned long long)hi << 32 | lo;
  }
};
using Key32 = Key<uint32_t>;
using Key64 = Key<unsigned long long>;

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float warp_most(float v) { return Key32::value(Key32::most(Key32::of(v))); }

// e^x for x <= 0 to 1e-15: x = n ln 2 + r with |r| <= 0.35, the series of e^r up to r^12 / 12!
// (the next term is below 2e-16), and 2^n in two factors, so that small results are denormal
// as they should be. exp() of the library decides the same and takes twice the instructions.
__device__ __forceinline__ double exp_down(double x) {
  x = fmax(x, -746.0);
  const double n = rint(x * 1.4426950408889634);
  const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));
  double y = 1.0 / 479001600.0;
  y = fma(y, r, 1.0 / 39916800.0);
  y = fma(y, r, 1.0 / 3628800.0);
  y = fma(y, r, 1.0 / 362880.0);
  y = fma(y, r, 1.0 / 40320.0);
  y = fma(y, r, 1.0 / 5040.0);
  y = fma(y, r, 1.0 / 720.0);
  y = fma(y, r, 1.0 / 120.0);
  y = fma(y, r, 1.0 / 24.0);
  y = fma(y, r, 1.0 / 6.0);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.0);
  y = fma(y, r, 1.0);
  const int k = (int)n, half = k / 2;
  const auto power = [](int i) { return __longlong_as_double((long long)(i + 1023) << 52); };
  return y * power(half) * power(k - half);
}
// A score in 64 bits, softmax's up to the factor 1 / (sum over the experts).
__device__ __forceinline__ double score_64(float l, int sigmoid, float most) {
  if (!sigmoid) return exp_down((double)l - (double)most);
  const double e = exp_down(-fabs((double)l)), r = __drcp_rn(1.0 + e);
  return l < 0.0f ? e * r : r;
}

// The score's sum with the bias, each rounded for itself: where the bias is so large that it
// decides by rounding, scores that differ less than that are one.
__device__ __forceinline__ double biased(double score, float bias) { return __dadd_rn(score, (double)bias); }

// The weights of a token's chosen experts: lane j has slot j's logit.
__device__ __forceinline__ float weight_of(float l, bool valid, float most, float total, int sigmoid, int renorm, float scale) {
  float s;
  if (!renorm) {
    s = sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - most) / total;
  } else if (sigmoid) {
    // s_i up to a common factor: e^min(l, 0) / (1 + e^-|l|)
    const float m = fminf(warp_most(valid ? l : -INFINITY), 0.0f);
    s = valid ? expf(fminf(l, 0.0f) - m) / (1.0f + expf(-fabsf(l))) : 0.0f;
    s = s / warp_sum(s);
  } else {
    const float m = warp_most(valid ? l : -INFINITY);
    s = valid ? expf(l - m) : 0.0f;
    s = s / warp_sum(s);
  }
  return valid ? s * scale : 0.0f;
}

// The two largest of keys seen so far.
template <typename K>
struct Best {
  K one = Key<K>::kNone, two = Key<K>::kNone;
  __device__ __forceinline__ void add(K k) {
    two = max(two, min(one, k));
    one = max(one, k);
  }
  __device__ __forceinline__ void add(const Best& o) {
    two = max(max(two, o.two), min(one, o.one));
    one = max(one, o.one);
  }
};

// Puts kNone in the place of the keys whose groups do not stay. Lane i holds experts i P
// .. + P. `worth`: a key's score (plus bias), which group values are sums of. `values`: the
// warp's place for its groups' values.
template <int P, typename K, typename F>
__device__ __forceinline__ void keep_groups(const RouteArgs& a, K (&key)[P], unsigned long long* values, F worth) {
  const int lane = threadIdx.x & 31, first = lane * P, size = a.E / a.groups, lanes = size / P;
  const auto value_of = [&](const Best<K>& b) -> unsigned long long {
    if (a.best == 1 || b.one == Key<K>::kNone) return b.one == Key<K>::kNone ? 0 : b.one;
    return Key64::of(worth(b.one) + (b.two != Key<K>::kNone ? worth(b.two) : 0.0));
  };
  if (size == lanes * P && (lanes & (lanes - 1)) == 0 && lanes >= 1) {
    // a group is `lanes` lanes
    Best<K> b;
#pragma unroll
    for (int p = 0; p < P; ++p) b.add(key[p]);
    for (int d = 1; d < lanes; d *= 2) {
      Best<K> o;
      o.one = __shfl_xor_sync(0xffffffffu, b.one, d);
      o.two = __shfl_xor_sync(0xffffffffu, b.two, d);
      b.add(o);
    }
    const unsigned long long mine = value_of(b);
    const int g = lane / lanes;
    int ahead = 0;
    for (int o = 0; o < a.groups; ++o) {
      const unsigned long long other = __shfl_sync(0xffffffffu, mine, o * lanes);
      ahead += other > mine || (other == mine && o < g);
    }
    if (ahead >= a.top_groups) {
#pragma unroll
      for (int p = 0; p < P; ++p) key[p] = Key<K>::kNone;
    }
    return;
  }
  for (int g = 0; g < a.groups; ++g) {
    Best<K> b;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (first + p >= g * size && first + p < (g + 1) * size) b.add(key[p]);
    const K one = Key<K>::most(b.one);
    const int holder = __ffs(__ballot_sync(0xffffffffu, b.one == one)) - 1;
    b.two = Key<K>::most(lane == holder ? b.two : b.one);
    b.one = one;
    if (lane == 0) values[g] = value_of(b);
  }
  __syncwarp();
  // a lane a group: does it stay? Said in the value's last place, once all are read.
  constexpr int kMost = kMaxExperts / 32;
  uint32_t stays = 0;
  for (int i = 0; i < kMost && i * 32 < a.groups; ++i) {
    const int g = i * 32 + lane;
    if (g >= a.groups) break;
    const unsigned long long mine = values[g];
    int ahead = 0;
    for (int o = 0; o < a.groups; ++o) ahead += values[o] > mine || (values[o] == mine && o < g);
    stays |= (uint32_t)(ahead < a.top_groups) << i;
  }
  __syncwarp();
  for (int i = 0; i < kMost && i * 32 + lane < a.groups; ++i) values[i * 32 + lane] = stays >> i & 1;
  __syncwarp();
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (first + p < a.E && !values[(first + p) / size]) key[p] = Key<K>::kNone;
  __syncwarp();
}

// The expert of slot `lane`: one choice after the other, the largest key, its lowest index.
// This lane holds experts first, first + 1, ..., later lanes later ones.
template <int P, typename K>
__device__ __forceinline__ int choose(int top, K (&key)[P], int first) {
  const int lane = threadIdx.x & 31;
  K mine = Key<K>::kNone;
#pragma unroll
  for (int p = 0; p < P; ++p) mine = max(mine, key[p]);
  int id = -1;
  for (int j = 0; j < top; ++j) {
    const K k = Key<K>::most(mine);
    if (k == Key<K>::kNone) break;
    const int from = __ffs(__ballot_sync(0xffffffffu, mine == k)) - 1;
    int e = first;
    if (lane == from) {  // it gives its first such key and looks for its next
      bool given = false;
      mine = Key<K>::kNone;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (!given && key[p] == k) key[p] = Key<K>::kNone, given = true, e = first + p;
        mine = max(mine, key[p]);
      }
    }
    e = __shfl_sync(0xffffffffu, e, from);
    if (lane == j) id = e;
  }
  return id;
}

// The choice with every key in 64 bits (or, without a bias, of logits): the expert of slot
// `lane`. For the tokens that route_token's shorter way does not decide.
template <typename T, int P>
__device__ __noinline__ int choose_long(const RouteArgs& a, const T* logits, float most, unsigned long long* values) {
  const int first = (threadIdx.x & 31) * P;
  float l[P];
#pragma unroll
  for (int p = 0; p < P; ++p) l[p] = first + p < a.E ? to_f32(logits[first + p]) : -INFINITY;
  if (!a.bias) {
    uint32_t key[P];
#pragma unroll
    for (int p = 0; p < P; ++p) key[p] = Key32::of(l[p]);
    if (a.groups > 1) keep_groups<P>(a, key, values, [&](uint32_t k) { return score_64(Key32::value(k), a.sigmoid, most); });
    return choose<P>(a.top, key, first);
  }
  unsigned long long key[P];
  double s[P], over = 1.0;
#pragma unroll
  for (int p = 0; p < P; ++p) s[p] = score_64(l[p], a.sigmoid, most);
  if (!a.sigmoid) {
    over = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) over += s[p];
    over = __drcp_rn(warp_sum(over));
  }
#pragma unroll
  for (int p = 0; p < P; ++p) key[p] = l[p] == -INFINITY ? Key64::kNone : Key64::of(biased(s[p] * over, a.bias[first + p]));
  if (a.groups > 1) keep_groups<P>(a, key, values, [](unsigned long long k) { return Key64::value(k); });
  return choose<P>(a.top, key, first);
}

// A score for the choice, with the approximate exponential (2^-22 of itself) and reciprocal
// (2^-23). With x its argument, whose product with log2 e and that constant are rounded, the
// exponential is off by (2 + 1.2 |x|) 2^-23 of itself. A sigmoid s moves by s (1 - s) as much, where
// s (1 - s) |x| <= 0.23, and by 1.5 2^-23 of itself for the sum and the reciprocal: 2.3 2^-23 in all. A
// probability p = e^-D / total moves by (2 + 1.7 D) 2^-23 of itself, where D p <= 0.4 pmax, and with
// its total, which is off by 34 2^-23 of itself (the mean of D is below ln E, and 37 additions).
__device__ __forceinline__ float quick_exp(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504f));
  return y;
}
__device__ __forceinline__ float quick_score(float l, int sigmoid, float most, float part) {
  if (!sigmoid) return quick_exp(l - most) * part;
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + quick_exp(-l)));
  return y;
}
// How far a key in 32 bits may then be from its 64-bit value, with the rounding of its sum
// with a bias of up to bmax. pmax is `part`.
__device__ __forceinline__ float key_bound(int sigmoid, float part, float bmax) { return (sigmoid ? 0x1p-21f : 0x1p-17f * part) + 0x1p-23f * bmax; }

// softmax's 1 / (sum over the experts) in 64 bits, for score_64; 1 for sigmoid.
template <typename T>
__device__ __noinline__ double over_of(const RouteArgs& a, const T* logits, int first, int per, float most) {
  if (a.sigmoid) return 1.0;
  double sum = 0.0;
#pragma unroll 1
  for (int e = first; e < first + per; ++e) sum += score_64(to_f32(logits[e]), 0, most);
  return __drcp_rn(warp_sum(sum));
}

// A token by a warp. A group lies on a.lanes lanes, a power of two, each with a.each of its
// experts or fewer, P at most; where there are more groups than lanes all experts lie so as one
// (a.cut). `vec`: rows of logits on 16 bytes.
//
// Without a bias keys are logits, and exact. With one they are 32-bit at first, off by `off`.
// At least `top` of them are no less than the top-th largest of the lanes' largest, so
// those that are, or are 2 off below, ten or so, are all that the choice can turn on: a lane
// each, ranked by comparing each with all, and where two are within 2 off in 64 bits (a few
// tokens of a thousand). Groups are compared likewise. With more candidates than lanes, or
// groups, choose_long. One choice after the other with all keys in
// 64 bits took 30 us for 8192 tokens of 256 experts, a third of it 64-bit arithmetic; this 13.
// Its 1150 instructions a token fill 8.1 us of issue slots; the rest is latency that 42 % of the
// warps (64 registers a thread) do not hide.
template <typename T, int P>
__device__ __forceinline__ void route_token(const RouteArgs& a, int64_t t, unsigned long long* values, int* candidates, bool vec) {
  const int lane = threadIdx.x & 31, size = a.E / a.cut, g = lane / a.lanes, from = lane % a.lanes * a.each;
  const int first = g * size + from, own = g < a.cut ? min(size - from, a.each) : 0;  // (own may be below 0)
  const T* logits = static_cast<const T*>(a.logits) + t * a.E;
  float l[P];
  if (vec && P * sizeof(T) >= 16 && a.each == P && own == P && first % P == 0) {
    constexpr int kEach = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < P / kEach; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(logits + first)[i];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if constexpr (sizeof(T) == 4)
          l[i * kEach + j] = __uint_as_float(w[j]);
        else
          l[i * kEach + j] = j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
      }
    }
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) l[p] = p < own ? to_f32(logits[first + p]) : -INFINITY;
  }
  float b[P], bmax = 0.0f;
  bool bad = false;
  if (a.bias) {
    if (reinterpret_cast<uintptr_t>(a.bias) % 16 == 0 && P >= 4 && own == P && first % 4 == 0) {
#pragma unroll
      for (int i = 0; i < P / 4; ++i) {
        const float4 f = reinterpret_cast<const float4*>(a.bias + first)[i];
        b[4 * i] = f.x, b[4 * i + 1] = f.y, b[4 * i + 2] = f.z, b[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int p = 0; p < P; ++p) b[p] = p < own ? a.bias[first + p] : 0.0f;
    }
    // the largest magnitude, by its bits: a NaN is above infinity
    uint32_t bits = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) bits = max(bits, __float_as_uint(b[p]) & 0x7fffffffu);
    bits = __reduce_max_sync(0xffffffffu, bits);
    bad = bits > 0x7f800000u;
    if (bits == 0x7f800000u) {  // of the finite ones
      bits = 0;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (fabsf(b[p]) < INFINITY) bits = max(bits, __float_as_uint(b[p]) & 0x7fffffffu);
      bits = __reduce_max_sync(0xffffffffu, bits);
    }
    bmax = __uint_as_float(bits);
  }
  const bool live = !a.live || a.live[t];
  float most = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    bad |= isnan(l[p]);
    most = fmaxf(most, l[p]);
  }
  most = warp_most(most);
  bad = __any_sync(0xffffffffu, bad || (!a.sigmoid && most == INFINITY));
  int* ids = a.ids + t * a.top;
  float* weights = a.weights + t * a.top;
  if (bad || !live || most == -INFINITY) {
    if (lane < a.top) {
      ids[lane] = -1;
      weights[lane] = bad && live ? NAN : 0.0f;
    }
    return;
  }
  const bool sums = a.groups > 1 && a.best > 1;  // group values are sums of scores
  float total = 1.0f, part = 1.0f, off = 0.0f;
  if (!a.sigmoid && (a.bias || sums || !a.renorm)) {
    total = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) total += a.renorm ? quick_exp(l[p] - most) : expf(l[p] - most);
    total = warp_sum(total);
    part = 1.0f / total;
  }
  if (a.bias || sums) off = key_bound(a.sigmoid, part, bmax);
  uint32_t key[P];
  if (!a.bias) {
#pragma unroll
    for (int p = 0; p < P; ++p) key[p] = Key32::of(l[p]);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) key[p] = l[p] == -INFINITY ? Key32::kNone : Key32::of(quick_score(l[p], a.sigmoid, most, part) + b[p]);
  }
  bool sure = true;
  if (a.groups > 1) {
    const int lanes = a.lanes;
    sure = a.cut == a.groups;
    if (sure) {
      Best<uint32_t> best;
#pragma unroll
      for (int p = 0; p < P; ++p) best.add(key[p]);
      for (int d = 1; d < lanes; d *= 2) {
        Best<uint32_t> o;
        o.one = __shfl_xor_sync(0xffffffffu, best.one, d);
        o.two = __shfl_xor_sync(0xffffffffu, best.two, d);
        best.add(o);
      }
      uint32_t mine = best.one;
      if (sums && mine != Key32::kNone) {
        const auto worth = [&](uint32_t k) { return a.bias ? Key32::value(k) : quick_score(Key32::value(k), a.sigmoid, most, part); };
        mine = Key32::of(worth(best.one) + (best.two != Key32::kNone ? worth(best.two) : 0.0f));
      }
      int ahead = 0;
      for (int o = 0; o < a.groups; ++o) {
        const uint32_t other = __shfl_sync(0xffffffffu, mine, o * lanes);
        ahead += other > mine || (other == mine && o < g);
      }
      bool stays = ahead < a.top_groups;
      if (a.bias || sums) {
        // a sum of two is off by twice as much, and by its own rounding
        const uint32_t kept = __reduce_min_sync(0xffffffffu, stays ? mine : 0xffffffffu);
        const uint32_t dropped = __reduce_max_sync(0xffffffffu, stays || g >= a.groups ? Key32::kNone : mine);
        if (dropped != Key32::kNone && Key32::value(kept) - Key32::value(dropped) <= 5.0f * off) {
          // the keys that may be a group's best, in 64 bits, and the groups compared so
          const uint32_t last = sums ? best.two : best.one;
          const uint32_t least = last == Key32::kNone ? last + 1 : Key32::of(Key32::value(last) - (a.bias ? 2.0f * off : 0.0f));
          uint32_t which = 0;
#pragma unroll
          for (int p = 0; p < P; ++p) which |= (uint32_t)(key[p] >= least && key[p] != Key32::kNone) << p;
          const double over = a.bias ? over_of(a, logits, first, own, most) : 1.0;
          Best<unsigned long long> wide;
          while (__any_sync(0xffffffffu, which)) {
            if (which) {
              const int e = first + __ffs(which) - 1;
              const float x = to_f32(logits[e]);
              wide.add(Key64::of(a.bias ? biased(score_64(x, a.sigmoid, most) * over, a.bias[e]) : (double)x));
              which &= which - 1;
            }
          }
          for (int d = 1; d < lanes; d *= 2) {
            Best<unsigned long long> o;
            o.one = __shfl_xor_sync(0xffffffffu, wide.one, d);
            o.two = __shfl_xor_sync(0xffffffffu, wide.two, d);
            wide.add(o);
          }
          unsigned long long value = wide.one;
          if (sums && value != Key64::kNone) {
            const auto worth = [&](unsigned long long k) { return a.bias ? Key64::value(k) : score_64((float)Key64::value(k), a.sigmoid, most); };
            value = Key64::of(worth(wide.one) + (wide.two != Key64::kNone ? worth(wide.two) : 0.0));
          }
          ahead = 0;
          for (int o = 0; o < a.groups; ++o) {
            const unsigned long long other = __shfl_sync(0xffffffffu, value, o * lanes);
            ahead += other > value || (other == value && o < g);
          }
          stays = ahead < a.top_groups;
        }
      }
      if (!stays) {
#pragma unroll
        for (int p = 0; p < P; ++p) key[p] = Key32::kNone;
      }
    }
  }
  int id = -1, place = lane, count = 0;
  if (sure && !a.bias) {  // keys are exact
    id = choose<P>(a.top, key, first);
    count = __popc(__ballot_sync(0xffffffffu, id >= 0));
  } else if (sure) {
    // The top-th largest of the lanes' largest, or (equal ones go together) a lower one.
    uint32_t left = Key32::kNone, least = Key32::kNone;
#pragma unroll
    for (int p = 0; p < P; ++p) left = max(left, key[p]);
    for (int j = 0; j < a.top; ++j) {
      least = Key32::most(left);
      if (left == least) left = Key32::kNone;
    }
    if (least != Key32::kNone) least = Key32::of(Key32::value(least) - 2.0f * off);
    least = max(least, Key32::kNone + 1);
    int mine = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) mine += key[p] >= least;
    int before = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += o;
    }
    count = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    sure = count <= 32;
    if (sure) {
      // candidate i is lane i's, by rising index
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (key[p] >= least) {
          candidates[before] = first + p;
          candidates[32 + before++] = (int)key[p];
        }
      __syncwarp();
      if (lane < count) id = candidates[lane];
      const uint32_t k = lane < count ? (uint32_t)candidates[32 + lane] : Key32::kNone;
      __syncwarp();
      const float chosen = id >= 0 ? to_f32(logits[id]) : -INFINITY, bias = id >= 0 ? a.bias[id] : 0.0f, value = Key32::value(k);
      place = 0;
      bool close = false;
      for (int o = 0; o < count; ++o) {
        const uint32_t other = __shfl_sync(0xffffffffu, k, o);
        place += other > k || (other == k && o < lane);
        close |= fabsf(Key32::value(other) - value) <= 2.0f * off && o != lane;
      }
      if (__any_sync(0xffffffffu, close && id >= 0)) {
        const double over = over_of(a, logits, first, own, most);
        const unsigned long long wide = id >= 0 ? Key64::of(biased(score_64(chosen, a.sigmoid, most) * over, bias)) : Key64::kNone;
        place = 0;
        for (int o = 0; o < count; ++o) {
          const unsigned long long other = __shfl_sync(0xffffffffu, wide, o);
          place += other > wide || (other == wide && o < lane);
        }
      }
      if (place >= a.top) id = -1;
    }
  }
  if (!sure) {
    id = choose_long<T, P>(a, logits, most, values);
    place = lane;
    count = __popc(__ballot_sync(0xffffffffu, id >= 0));
  }
  const float chosen = id >= 0 ? to_f32(logits[id]) : -INFINITY;
  const float w = weight_of(chosen, id >= 0, most, total, a.sigmoid, a.renorm, a.scale);
  if (id >= 0) {
    ids[place] = id;
    weights[place] = w;
  }
  if (lane >= count && lane < a.top) {  // fewer than asked for
    ids[lane] = -1;
    weights[lane] = 0.0f;
  }
}

// ── the rows' order ─────────────────────────────────────────────────────────
// A counting sort by a cluster. Each warp has a run of slots and a counter for each expert;
// the counters' prefix sums over warps, then over CTAs (whose totals the others
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
static size_t order_shared(int E) { return sizeof(int) * ((kOrderWarps + 2) * (size_t)E + 32); }

// The CTA's slots are lo .. hi. Several clusters (`parts`) may do this at once: each counts
// all slots, and places the `part`-th share of every warp's.
__device__ __forceinline__ void order_rows(const OrderArgs& a, int* shared, int64_t lo, int64_t hi, int part, int parts) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int E = a.E, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  int* count = shared;                   // [warp][expert]
  int* total = count + kOrderWarps * E;  // this CTA's rows of each expert
  int* start = total + E;                // the first row of each expert that is this CTA's
  int* sums = start + E;                 // [32] of the scan, and the number of rows
  const int64_t per = ((hi - lo + 31) / 32 + kOrderWarps - 1) / kOrderWarps * 32;
  const int64_t from = min(hi, lo + warp * per), to = min(hi, from + per);
  int* mine = count + warp * E;
  for (int i = lane; i < E; i += 32) mine[i] = 0;
  __syncwarp();
  constexpr int kAhead = 8;  // loads in flight
  for (int64_t s = from; s < to; s += 32 * kAhead) {
    int id[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) id[i] = s + i * 32 + lane < to ? a.ids[s + i * 32 + lane] : -1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if ((unsigned)id[i] < (unsigned)E) atomicAdd(mine + id[i], 1);
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < E) {
    int run = 0;
#pragma unroll 8
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
#pragma unroll 8
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
    if (rank == 0 && part == 0) {
      a.offsets[e] = first;
      if (e == E - 1) a.offsets[E] = rows;
    }
  }
  cluster.sync();  // nobody leaves while its totals are read
  const int64_t steps = (to - from + 31) / 32, begin = from + steps * part / parts * 32, end = min(to, from + steps * (part + 1) / parts * 32);
  for (int64_t s = from; s < begin; s += 32 * kAhead) {  // the shares before
    int id[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) id[i] = s + i * 32 < begin ? a.ids[s + i * 32 + lane] : -1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if ((unsigned)id[i] < (unsigned)E) atomicAdd(mine + id[i], 1);
  }
  __syncwarp();
  for (int64_t s = begin; s < end; s += 32 * kAhead) {
    int id[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) id[i] = s + i * 32 + lane < end ? a.ids[s + i * 32 + lane] : -1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t slot = s + i * 32 + lane;
      if (slot - lane >= end) break;
      const bool valid = (unsigned)id[i] < (unsigned)E;
      const unsigned peers = __match_any_sync(0xffffffffu, valid ? id[i] : -1), below = peers & ((1u << lane) - 1);
      if (valid) {
        const int at = start[id[i]] + mine[id[i]] + __popc(below);
        a.rows_of[at] = (int)((uint32_t)slot / (uint32_t)a.top);
        a.row_at[slot] = at;
      } else if (slot < end) {
        a.row_at[slot] = -1;
      }
      __syncwarp();
      if (valid && below == 0) mine[id[i]] += __popc(peers);
      __syncwarp();
    }
  }
  for (int64_t r = rows + ((int64_t)part * ctas + rank) * blockDim.x + threadIdx.x; r < a.n; r += (int64_t)parts * ctas * blockDim.x) a.rows_of[r] = -1;
}

// ── the kernels ─────────────────────────────────────────────────────────────
// The choice alone, four tokens a CTA.
template <typename T, int P>
__global__ void __launch_bounds__(128) route_kernel(RouteArgs a, bool vec) {
  extern __shared__ __align__(16) unsigned long long values[];  // of a warp's groups
  __shared__ int candidates[4][64];
  pdl_trigger();
  const int warp = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * 4 + warp;
  if (t < a.T) route_token<T, P>(a, t, values + warp * (a.groups > 1 ? a.groups : 0), candidates[warp], vec);
}
// The order alone, by one cluster, behind it.
__global__ void __launch_bounds__(kOrderWarps * 32) order_rows_kernel(OrderArgs a) {
  extern __shared__ __align__(16) int shared[];
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int64_t steps = (a.n + 31) / 32, per = (steps + cluster.num_blocks() - 1) / cluster.num_blocks() * 32;
  const int64_t lo = min(a.n, (int64_t)cluster.block_rank() * per), hi = min(a.n, lo + per);
  pdl_wait();
  order_rows(a, shared, lo, hi, blockIdx.x / cluster.num_blocks(), gridDim.x / cluster.num_blocks());
}
// Both by one cluster, for few tokens.
template <typename T, int P>
__global__ void __launch_bounds__(kOrderWarps * 32) route_and_order_kernel(RouteArgs a, OrderArgs o, bool vec) {
  extern __shared__ __align__(16) int shared[];
  __shared__ int candidates[kOrderWarps][64];
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int warp = threadIdx.x >> 5;
  unsigned long long* values = reinterpret_cast<unsigned long long*>(shared) + warp * (a.groups > 1 ? a.groups : 0);
  const int64_t per = (a.T + cluster.num_blocks() - 1) / cluster.num_blocks();
  const int64_t lo = min(a.T, (int64_t)cluster.block_rank() * per), hi = min(a.T, lo + per);
  for (int64_t t = lo + warp; t < hi; t += kOrderWarps) route_token<T, P>(a, t, values, candidates[warp], vec);
  __syncthreads();  // the ids are this CTA's own
  order_rows(o, shared, lo * a.top, hi * a.top, 0, 1);
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
  // a token without experts has no gradient, whatever its logits hold
  const bool dense = !a.sigmoid && !a.renorm && __any_sync(0xffffffffu, valid);
  if (dense) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int e = i * 32 + lane;
      p[i] = e < E ? to_f32(logits[e]) : -INFINITY;
      most = fmaxf(most, p[i]);
    }
    most = warp_most(most);
    if (most == -INFINITY) most = 0.0f;  // every expert masked: all of p is 0
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) total += p[i] = expf(p[i] - most);
    total = warp_sum(total);
    if (total == 0.0f) total = 1.0f;
  }
  const float u = weight_of(l, valid, most, total, a.sigmoid, a.renorm, 1.0f);
  const float mean = a.sigmoid && !a.renorm ? 0.0f : warp_sum(g * u);
  __syncwarp();  // the row is read: dlogits may be the logits' own memory
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

constexpr int kRouteShared = 160 * 1024;  // more than order_shared() asks for, or 256 groups' values of every warp

template <typename... K, typename... A>
static cudaError_t cluster_launch(void (*kernel)(K...), unsigned ctas, unsigned clusters, size_t shared, bool behind, int device, unsigned long long* done, cudaStream_t st, A... args) {
  if (const cudaError_t e = allow_shared(kernel, kRouteShared, device, done)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * clusters);
  cfg.blockDim = dim3(kOrderWarps * 32);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = behind ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A direct call of up to this many tokens, where a lane has P experts at most, is one launch: one
// cluster chooses and orders, which spares the host more than the GPU loses. In microseconds a pass
// among others, one launch and two, over softmax and sigmoid, bias and groups: 128 tokens of 64
// experts 10.3 to 12.3 and 12.4, of 128 the same, 1 token of either 9.4 to 10.3 and 12.4; 16 tokens of
// 256 experts 10.3 to 12.3 and 12.4, but 32 in groups 14.2 and 12.4, 64 of 512 16.4 to 18.5 and 12.4,
// 64 of 1024 28.9 to 45 and 13.4 to 16.4 (their keys spill in a CTA of 1024 threads). The GPU alone
// always takes longer in one (64 tokens of 32 experts 7.9 us, 6.8 in two; 128 of 64 8.4 to 11.1, 7.0
// to 8.6), so a captured call, whose replays cost the host nothing, is two.
template <int P>
constexpr int64_t kFewTokens = P <= 4 ? 128 : P <= 8 ? 16 : 0;
// Else the order is made by clusters of eight CTAs, as many as a warp has steps of 32 slots,
// so that each places one or few (65536 slots 16.8 us by one cluster, 10.8 by eight).
constexpr unsigned kOrderCtas = 8, kOrderClusters = 8;

static bool captured(cudaStream_t st) {
  cudaStreamCaptureStatus status;
  if (cudaStreamIsCapturing(st, &status) == cudaSuccess) return status != cudaStreamCaptureStatusNone;
  cudaGetLastError();  // the launch will say so itself
  return false;
}

// `ordered`: the rows' order is made too.
template <typename T, int P>
static cudaError_t route_go(const RouteArgs& a, const OrderArgs* o, bool vec, int device, bool* ordered, cudaStream_t st) {
  const size_t values = a.groups > 1 ? sizeof(unsigned long long) * a.groups : 0;
  if constexpr (kFewTokens<P> > 0) {
    if (o && a.T > 0 && a.T <= kFewTokens<P> && !captured(st)) {
      static unsigned long long done;
      const unsigned ctas = (unsigned)std::min<int64_t>(kOrderCtas, (a.T + kOrderWarps - 1) / kOrderWarps);
      *ordered = true;
      return cluster_launch(route_and_order_kernel<T, P>, ctas, 1, std::max(order_shared(a.E), kOrderWarps * values), false, device, &done, st, a, *o, vec);
    }
  }
  if (a.T) route_kernel<T, P><<<(unsigned)((a.T + 3) / 4), 128, 4 * values, st>>>(a, vec);
  return cudaSuccess;
}
template <typename T>
static cudaError_t route_launch(RouteArgs a, const OrderArgs* o, bool vec, int device, bool* ordered, cudaStream_t st) {
  a.cut = a.groups;
  a.lanes = 1;
  while (a.lanes * 2 * a.cut <= 32) a.lanes *= 2;
  a.each = (a.E / a.cut + a.lanes - 1) / a.lanes;
  if (a.cut > 32 || a.each > 32) a.cut = 1, a.lanes = 32, a.each = (a.E + 31) / 32;
  const int most = std::max(a.each, (a.E + 31) / 32);  // of a lane, choose_long's among them
  if (most <= 1) return route_go<T, 1>(a, o, vec, device, ordered, st);
  if (most <= 2) return route_go<T, 2>(a, o, vec, device, ordered, st);
  if (most <= 4) return route_go<T, 4>(a, o, vec, device, ordered, st);
  if (most <= 8) return route_go<T, 8>(a, o, vec, device, ordered, st);
  if (most <= 16) return route_go<T, 16>(a, o, vec, device, ordered, st);
  return route_go<T, 32>(a, o, vec, device, ordered, st);
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
  const bool bf16 = la.a[15].i32, vec = la.a[5].ptr % 16 == 0 && (int64_t)a.E * (bf16 ? 2 : 4) % 16 == 0, ordering = given(la, 2);
  OrderArgs o = {};
  o.ids = a.ids;
  o.offsets = reinterpret_cast<int*>(la.a[2].ptr);
  o.rows_of = reinterpret_cast<int*>(la.a[3].ptr);
  o.row_at = reinterpret_cast<int*>(la.a[4].ptr);
  o.n = a.T * a.top;
  o.E = a.E;
  o.top = a.top;
  bool ordered = !ordering;
  cudaError_t e = bf16 ? route_launch<uint16_t>(a, ordering ? &o : nullptr, vec, la.device, &ordered, st)
                       : route_launch<float>(a, ordering ? &o : nullptr, vec, la.device, &ordered, st);
  if (e == cudaSuccess && !ordered) {
    static unsigned long long done;
    const unsigned ctas = a.T ? kOrderCtas : 1, clusters = (unsigned)std::max<int64_t>(1, std::min<int64_t>(kOrderClusters, o.n / (32 * kOrderWarps * ctas)));
    e = cluster_launch(order_rows_kernel, ctas, clusters, order_shared(a.E), a.T > 0, la.device, &done, st, o);
  }
  if (e != cudaSuccess) return fail(MTL_ERR_CUDA, "route_experts: %s", cudaGetErrorString(e));
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
