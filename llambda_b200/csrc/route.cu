// Choice of experts from router logits: softmax or sigmoid scores, a bias that
// only steers the choice, expert groups, top-k, renormalised weights.
//
// Mathematics, per token: s = softmax(l) or 1 / (1 + exp(-l)); c = s + bias;
// a group's score is its largest c or the sum of its two largest; experts
// outside the top_groups best groups are out; the top_k largest c are chosen,
// ties to the lowest index; weight = s (over the chosen ones' sum) * scale.
// An expert whose logit is -inf has score 0 and is chosen after all others.
//
// The choice has to be that of exact scores, and two experts' scores can lie
// closer than fp32 tells apart.  Where the order of the logits is the order of
// the choice (no bias, and no sums of two scores) the logits themselves are
// compared.  Elsewhere c is computed in fp32 first, and a token for which some
// comparison that decided was closer than the error of c is done again in fp64
// (well under 1 in 10 tokens for logits of unit variance).  Where that is too
// close too (scores next to 1, or beside large biases), the part of a choice that
// its double rounds off is kept beside it, and choices that are still equal go by
// their logits.  That pass is rare and the slowest: in the place of the fp64 one
// it took 8191 tokens with 256 experts in 8 groups from 17.4 to 24.9 us; behind
// it, with the checks that lead to it, 18.2.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "engine.cuh"
#include "kernels.h"

namespace lb {

namespace {

constexpr int kRouteWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

// Order-preserving maps of floats to unsigned keys: 0 is below every value (an
// expert that is out), 1 a NaN (chosen last), then -inf upwards; -0 equals +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (isnan(v)) return 1u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  if (isnan(v)) return 1ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k <= 1u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ double key_value(unsigned long long k) {
  if (k <= 1ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(kFull, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
  const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(v >> 32));
  const uint32_t lo =
      __reduce_max_sync(kFull, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (unsigned long long)hi << 32 | lo;
}

// The score of a logit; m is the largest logit and z the sum of exp(l - m)
// (softmax).  A row of -inf only scores 0.
__device__ __forceinline__ float score(const RouteParams& r, float l, float m, float z) {
  if (l == -INFINITY) return 0.0f;
  return r.softmax ? expf(l - m) / z : 1.0f / (1.0f + expf(-l));
}

// What the choice goes by, in fp32 (fast exp and division) and in fp64, errors
// within choice_error.
__device__ __forceinline__ float choice(const RouteParams& r, const float* bias, float l, float m,
                                        float z, int e) {
  if (l == -INFINITY) return l;
  const float s =
      r.softmax ? __fdividef(__expf(l - m), z) : __fdividef(1.0f, 1.0f + __expf(-l));
  return bias ? s + __ldg(bias + e) : s;
}
__device__ __forceinline__ double choice(const RouteParams& r, const float* bias, float l, float m,
                                         double z, int e) {
  if (l == -INFINITY) return (double)l;
  const double s = r.softmax ? exp((double)l - (double)m) / z : 1.0 / (1.0 + exp(-(double)l));
  return bias ? s + (double)__ldg(bias + e) : s;
}

// Bound on the error of the difference of two choices near c (half of it: of one
// choice, and of its part in a sum; z's error is common to all choices and changes
// no order).  fp32, sigmoid: __expf is off by (2 + 1.173 |l|) steps at most, which
// moves s by at most 0.63 steps of 2^-23, the sum by half a step, __fdividef by
// two.  Softmax, relative to the largest score smax = 1 / z: the exponentials and
// the division 5e-7 each, z (its exponentials and 37 additions) 4e-6.  Then the
// rounding of the sums with the bias.
__device__ __forceinline__ float choice_error(const RouteParams& r, float c, float smax) {
  return (r.softmax ? 8e-6f * smax : 1e-6f) + 2.5e-7f * fabsf(c);
}
// fp64: exp is off by a step, the sum and the division by half a step each.
__device__ __forceinline__ double choice_error(const RouteParams& r, double c, double smax) {
  return 2e-15 * smax + 5e-16 * fabs(c);
}

__device__ __forceinline__ float logit_at(const float* p, long i) { return __ldg(p + i); }
__device__ __forceinline__ float logit_at(const __nv_bfloat16* p, long i) {
  return __bfloat162float(p[i]);
}

// A choice in 64 bits as keys that compare in this order: the nearest double, the
// rest of the sum that it rounds (lo: as a float, so that sums of the same terms
// in another order compare equal), the logit.  All 0: an expert that is out.
struct Exact {
  unsigned long long k;
  uint32_t lo, l;
  double rest;
};
__device__ __forceinline__ bool operator>(const Exact& a, const Exact& b) {
  return a.k != b.k ? a.k > b.k : a.lo != b.lo ? a.lo > b.lo : a.l > b.l;
}
__device__ __forceinline__ bool operator==(const Exact& a, const Exact& b) {
  return a.k == b.k && a.lo == b.lo && a.l == b.l;
}
__device__ __forceinline__ void take_two(Exact& a, Exact& b, const Exact& v) {  // the two largest
  if (v > a)
    b = a, a = v;
  else if (v > b)
    b = v;
}
__device__ __forceinline__ Exact shfl(const Exact& v, int lane) {
  return {__shfl_sync(kFull, v.k, lane), __shfl_sync(kFull, v.lo, lane),
          __shfl_sync(kFull, v.l, lane), __shfl_sync(kFull, v.rest, lane)};
}
// The warp's largest, and the lowest lane that has it.
__device__ __forceinline__ Exact warp_max(const Exact& v, int& owner) {
  Exact r;
  r.k = warp_max(v.k);
  bool in = v.k == r.k;
  r.lo = warp_max(in ? v.lo : 0u);
  in = in && v.lo == r.lo;
  r.l = warp_max(in ? v.l : 0u);
  in = in && v.l == r.l;
  owner = __ffs(__ballot_sync(kFull, in)) - 1;
  r.rest = __shfl_sync(kFull, v.rest, owner);
  return r;
}
// a + b + c with |c| small beside the sum, or a, b doubles of any size (their sum
// and its error: Knuth, The Art of Computer Programming 2, 4.2.2), logit key l.
__device__ __forceinline__ Exact exact_sum(double a, double b, double c, uint32_t l) {
  const double s = a + b, t = s - a, e = ((a - (s - t)) + (b - t)) + c;
  const double hi = s + e;
  if (!isfinite(hi)) return {order_key(s + c), 0u, 0u, 0.0};
  const double rest = e - (hi - s);
  return {order_key(hi), order_key((float)rest), l, rest};
}
__device__ __forceinline__ Exact exact_choice(const RouteParams& r, const float* bias, float l,
                                              float m, double z, int e) {
  if (l == -INFINITY) return {order_key((double)l), 0u, 0u, 0.0};
  const double b = bias ? (double)__ldg(bias + e) : 0.0;
  if (r.softmax) return exact_sum(b, exp((double)l - (double)m) / z, 0.0, order_key(l));
  // a positive logit's score as 1 less what is left
  if (l > 0.0f) return exact_sum(1.0, b, -1.0 / (1.0 + exp((double)l)), order_key(l));
  return exact_sum(b, 1.0 / (1.0 + exp(-(double)l)), 0.0, order_key(l));
}

// Whether the groups (one a lane) that are close to each other have a true tie: their
// two largest choices (g1, g2; `keys`: all, R + 1 a lane) are of equal logits and
// biases, that is all choices near the first are, and all near the second.  Not
// inlined, as choose_exact is not: the registers they take would be the whole
// kernel's (8192 tokens, 1024 experts: 83 -> 90 us).
template <int R, typename T>
__device__ __noinline__ bool groups_tie(RouteParams r, const T* row, const float* bias,
                                        const unsigned long long* keys, unsigned long long g1,
                                        unsigned long long g2, double smax, bool close) {
  const int lane = threadIdx.x & 31;
  const unsigned near = __ballot_sync(kFull, close);
  const int any = __ffs(near) - 1;
  if (any < 0) return false;
  const unsigned long long k1 = __shfl_sync(kFull, g1, any), k2 = __shfl_sync(kFull, g2, any);
  if (!__all_sync(kFull, !close || (g1 == k1 && g2 == k2))) return false;
  const double t1 = key_value(k1), t2 = key_value(k2);
  const double from1 = t1 - choice_error(r, t1, smax), from2 = t2 - choice_error(r, t2, smax);
  const int size = r.experts / r.groups;
  uint32_t low[4] = {~0u, ~0u, ~0u, ~0u}, high[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
  for (int j = 0; j < R; ++j) {
    const int e = lane * R + j;
    const double v = key_value(keys[lane * (R + 1) + j]);  // (not a number where there is none)
    if (e >= r.experts || !(near >> (e / size) & 1u) || !(v >= from2)) continue;
    const bool first = v >= from1;
    const uint32_t kl = order_key(logit_at(row, e)), kb = bias ? order_key(__ldg(bias + e)) : 0u;
    low[0] = min(low[0], first ? kl : ~0u), high[0] = max(high[0], first ? kl : 0u);
    low[1] = min(low[1], first ? kb : ~0u), high[1] = max(high[1], first ? kb : 0u);
    low[2] = min(low[2], first ? ~0u : kl), high[2] = max(high[2], first ? 0u : kl);
    low[3] = min(low[3], first ? ~0u : kb), high[3] = max(high[3], first ? 0u : kb);
  }
  bool same = true;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    same = __reduce_min_sync(kFull, low[i]) >= warp_max(high[i]) && same;
  return same;
}

// The choice of one token by one warp: lane L holds experts L * R .. L * R +
// R - 1, so equal keys go to the lowest lane that has one, and to its lowest j.
// Rank i's expert goes to lane i.  Returns false when some comparison that
// decided was closer than the error of the choices (by_logit: there is none):
// that of two groups, of two ranks, or of the last rank with an expert that is not
// chosen.  Equal logits and biases (`row`: the token's logits) are a true tie, which
// the index decides.
//
// Each round takes the warp's largest key, one reduction over the lanes' own
// largest.  A lane knows its two largest; the keys themselves are in shared
// memory (`keys`, R + 1 a lane), where the whole warp looks for the place of the
// one taken among its lane's, and for that lane's next two when both are gone.
// At 8191 tokens, 256 experts in 8 groups, top 8: 27 us with the keys in
// registers and each lane looking through its own in every round, 20 looking
// only when both are gone, 18 so.
template <int R, typename F, typename T>
__device__ __forceinline__ bool choose(const RouteParams& r, const T* row, const float (&l)[R],
                                       const float* bias, bool by_logit, float m, F z, int lane,
                                       void* shared, int& sel) {
  using K = decltype(order_key(F(0)));
  K* keys = static_cast<K*>(shared);
  const bool check = !by_logit;
  const F smax = r.softmax ? F(1) / z : F(1);
  K key[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane * R + j;
    key[j] = e >= r.experts ? K(0)
             : by_logit     ? order_key((F)l[j])
                            : order_key(choice(r, bias, l[j], m, z, e));
  }
  bool sure = true;
  if (r.top_groups < r.groups) {
    const int size = r.experts / r.groups, span = size / R;
    K g1 = 0, g2 = 0;  // lane g: group g's two largest
    if (size % R == 0 && (span & (span - 1)) == 0) {  // whole lanes, a power of two of them
      K a = 0, b = 0;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        b = max(b, min(a, key[j]));
        a = max(a, key[j]);
      }
      for (int o = 1; o < span; o <<= 1) {
        const K a2 = __shfl_xor_sync(kFull, a, o), b2 = __shfl_xor_sync(kFull, b, o);
        b = max(min(a, a2), max(b, b2));
        a = max(a, a2);
      }
      g1 = __shfl_sync(kFull, a, lane * span & 31);
      g2 = __shfl_sync(kFull, b, lane * span & 31);
    } else {
      for (int g = 0; g < r.groups; ++g) {
        const int lo = g * size, hi = lo + size;
        K a = 0, b = 0;  // this lane's two largest
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const int e = lane * R + j;
          const K v = e >= lo && e < hi ? key[j] : K(0);
          b = max(b, min(a, v));
          a = max(a, v);
        }
        const K first = warp_max(a);
        const int owner = __ffs(__ballot_sync(kFull, a == first)) - 1;
        const K second = warp_max(lane == owner ? b : a);
        if (lane == g) g1 = first, g2 = second;
      }
    }
    K gkey = r.group_top == 2 ? order_key(key_value(g1) + key_value(g2)) : g1;
    if (lane >= r.groups) gkey = 0;
    int rank = 0;  // groups before this lane's: larger ones, and equal ones of lower index
    for (int g = 0; g < r.groups; ++g) {
      const K v = __shfl_sync(kFull, gkey, g);
      rank += v > gkey || (v == gkey && g < lane);
    }
    const bool is_group = lane < r.groups;
    const unsigned kept = __ballot_sync(kFull, is_group && rank < r.top_groups);
    if (check) {
      // Every group left out against every one kept.  A sum is off by what its
      // addends are, however small it is itself.  One with NaN, or with an expert
      // that is masked, is exact.
      const bool two = r.group_top == 2, keep = kept >> lane & 1u;
      const F sum = key_value(gkey), v1 = key_value(g1), v2 = two ? key_value(g2) : F(0);
      const bool exact = isnan(sum) || (isinf(sum) && sum < 0 && (isinf(v1) || isinf(v2)));
      const F lim = isinf(sum) ? F(0)
                               : F(0.5) * (choice_error(r, v1, smax) +
                                         (two ? choice_error(r, v2, smax) : F(0))) +
                                     (sizeof(F) == 4 ? F(1.2e-7) : F(2.3e-16)) * fabs(sum);
      const K most = warp_max(is_group && !keep && !exact ? order_key(sum + lim) : K(0));
      const K least = warp_max(is_group && keep ? order_key(lim - sum) : K(0));
      if (most != 0 && key_value(most) >= -key_value(least)) {
        sure = false;
        if constexpr (sizeof(F) == 8) {
#pragma unroll
          for (int j = 0; j < R; ++j) keys[lane * (R + 1) + j] = key[j];
          sure = groups_tie<R>(r, row, bias, keys, g1, two ? g2 : g1, smax,
                               is_group && (keep ? sum - lim <= key_value(most)
                                                 : !exact && sum + lim >= -key_value(least)));
        }
      }
    }
    int g = lane * R / size, left = (g + 1) * size - lane * R;  // experts left in group g
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (!(kept >> (g & 31) & 1u)) key[j] = 0;
      if (--left == 0) ++g, left = size;
    }
  }
  K a = 0, b = 0, mine = 0, next = 0;  // mine: rank `lane`'s key; next: the best not chosen
#pragma unroll
  for (int j = 0; j < R; ++j) {
    b = max(b, min(a, key[j]));
    a = max(a, key[j]);
    keys[lane * (R + 1) + j] = key[j];
  }
  __syncwarp();
  for (int i = 0; i <= r.top_k; ++i) {
    if (i == r.top_k && !check) break;
    const K best = warp_max(a);
    if (best == 0) break;  // no expert left to compare with
    const int owner = __ffs(__ballot_sync(kFull, a == best)) - 1;
    // lane j: the owner's key j
    K v = lane < R ? keys[owner * (R + 1) + lane] : K(0);
    const int at = __ffs(__ballot_sync(kFull, v == best)) - 1;
    const int e = owner * R + at;
    if (i == r.top_k) {
      next = best;
      break;
    }
    if (lane == i) sel = e, mine = best;
    if (lane == at) {
      keys[owner * (R + 1) + at] = 0;
      v = 0;
    }
    const bool held = lane == owner;
    if (held) a = b, b = 0;
    if (R > 2 && __any_sync(kFull, held && a == 0)) {
      const K first = warp_max(v);
      const int one = __ffs(__ballot_sync(kFull, v == first)) - 1;
      const K second = warp_max(lane == one ? K(0) : v);
      if (held) a = first, b = second;
    }
    __syncwarp();
  }
  if (check) {
    const K after = __shfl_down_sync(kFull, mine, 1);
    const F c = key_value(mine), lim = choice_error(r, c, smax);
    const bool tied = lane < r.top_k - 1 && c - key_value(after) <= lim;
    if (__any_sync(kFull, tied)) {
      const float lv = logit_at(row, sel), bv = bias ? __ldg(bias + sel) : 0.0f;
      const float ln = __shfl_down_sync(kFull, lv, 1), bn = __shfl_down_sync(kFull, bv, 1);
      if (__any_sync(kFull, tied && (lv != ln || bv != bn))) sure = false;
    }
    const F last = __shfl_sync(kFull, c, r.top_k - 1);
    const F least = __shfl_sync(kFull, lim, r.top_k - 1);
    if (next != 0 && last - key_value(next) <= least) {
      const int e0 = __shfl_sync(kFull, sel, r.top_k - 1);
      const float l0 = logit_at(row, e0), b0 = bias ? __ldg(bias + e0) : 0.0f;
      bool near = false;
#pragma unroll 1
      for (int j = 0; j < R; ++j) {  // the keys of experts that are out or chosen are 0
        const K v = keys[lane * (R + 1) + j];
        if (v == 0 || !(last - key_value(v) <= least)) continue;
        const int e = lane * R + j;
        near |= logit_at(row, e) != l0 || (bias && __ldg(bias + e) != b0);
      }
      if (__any_sync(kFull, near)) sure = false;
    }
  }
  return sure;
}

// The choice by Exact keys; `shared` holds which experts are out (of lane i the bits of
// its R), the keys are worked out anew where they are looked at.
template <int R, typename T>
__device__ __noinline__ int choose_exact(RouteParams r, const T* row, const float* bias,
                                         float m, double z, void* shared) {
  const int lane = threadIdx.x & 31;
  int sel = 0;
  uint32_t* out = static_cast<uint32_t*>(shared);
  constexpr Exact kOut{0ull, 0u, 0u, 0.0};
  auto at = [&](int owner, int j) {  // expert owner * R + j
    const int e = owner * R + j;
    if (e >= r.experts || (out[owner] >> j & 1u)) return kOut;
    return exact_choice(r, bias, logit_at(row, e), m, z, e);
  };
  out[lane] = 0u;
  Exact a = kOut, b = kOut;
#pragma unroll(R < 4 ? R : 4)
  for (int j = 0; j < R; ++j) take_two(a, b, at(lane, j));
  if (r.top_groups < r.groups) {
    const int size = r.experts / r.groups, span = size / R;
    Exact g1 = kOut, g2 = kOut;  // lane g: group g's two largest
    if (size % R == 0 && (span & (span - 1)) == 0) {
      for (int o = 1; o < span; o <<= 1) {
        const Exact a2 = shfl(a, lane ^ o), b2 = shfl(b, lane ^ o);
        take_two(a, b, a2);
        take_two(a, b, b2);
      }
      g1 = shfl(a, lane * span & 31), g2 = shfl(b, lane * span & 31);
    } else {
      for (int g = 0; g < r.groups; ++g) {
        const int lo = max(g * size - lane * R, 0), hi = min((g + 1) * size - lane * R, R);
        a = b = kOut;
        for (int j = lo; j < hi; ++j) take_two(a, b, at(lane, j));
        int owner, other;
        const Exact first = warp_max(a, owner);
        const Exact second = warp_max(lane == owner ? b : a, other);
        if (lane == g) g1 = first, g2 = second;
      }
    }
    Exact rank_by = g1;
    if (r.group_top == 2) {
      const double d1 = key_value(g1.k), d2 = key_value(g2.k);
      rank_by = exact_sum(d1, d2, g1.rest + g2.rest, 0u);
    }
    if (lane >= r.groups) rank_by = kOut;
    int rank = 0;
    for (int g = 0; g < r.groups; ++g) {
      const Exact v = shfl(rank_by, g);
      rank += v > rank_by || (v == rank_by && g < lane);
    }
    const unsigned kept = __ballot_sync(kFull, lane < r.groups && rank < r.top_groups);
    a = kOut;
    for (int j = 0; j < R; ++j) {
      if (!(kept >> ((lane * R + j) / size & 31) & 1u)) out[lane] |= 1u << j;
      const Exact v = at(lane, j);
      if (v > a) a = v;
    }
  }
  __syncwarp();
  for (int i = 0; i < r.top_k; ++i) {
    int owner, one;
    const Exact best = warp_max(a, owner);
    Exact v = lane < R ? at(owner, lane) : kOut;  // lane j: the owner's j-th
    const int j = __ffs(__ballot_sync(kFull, v == best && lane < R)) - 1;
    if (lane == i) sel = owner * R + j;
    if (lane == j) {
      out[owner] |= 1u << j;
      v = kOut;
    }
    const Exact next = warp_max(v, one);
    if (lane == owner) a = next;
    __syncwarp();
  }
  return sel;
}

// Lane i: the weight of rank i, whose logit is l, in fp64 and relative to the
// largest chosen score: for tokens some of whose chosen scores are next to what
// fp32 can hold, or below it, although their shares are not.
__device__ __noinline__ float faint_weight(RouteParams r, float l, float m, float z) {
  const bool on = (threadIdx.x & 31) < r.top_k;
  const double top = key_value(warp_max(on ? order_key(l) : 0u));
  double s = 0.0;
  if (on && l != -INFINITY) {
    const double x = (double)l;
    if (r.softmax)
      s = r.renormalise ? exp(x - top) : exp(x - (double)m) / (double)z;
    else if (l > 0.0f)
      s = 1.0 / (1.0 + exp(-x));
    else
      s = exp(x - (r.renormalise ? fmin(top, 0.0) : 0.0)) / (1.0 + exp(x));
  }
  if (r.renormalise) {
    double sum = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    s /= sum;
  }
  return (float)(s * (double)r.scale);
}

// R consecutive logits, in the widest loads their size allows when the rows are aligned.
template <int R>
__device__ __forceinline__ void load_logits(const float* p, float (&l)[R]) {
  if constexpr (R >= 4) {
#pragma unroll
    for (int j = 0; j < R; j += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + j));
      l[j] = v.x, l[j + 1] = v.y, l[j + 2] = v.z, l[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) l[j] = __ldg(p + j);
  }
}
template <int R>
__device__ __forceinline__ void load_logits(const __nv_bfloat16* p, float (&l)[R]) {
  if constexpr (R >= 8) {
#pragma unroll
    for (int j = 0; j < R; j += 8) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + j));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        l[j + 2 * i] = __uint_as_float(w[i] << 16);
        l[j + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) l[j] = __bfloat162float(p[j]);
  }
}

// One warp per token.  vec: every row starts on 16 bytes.  The rare passes' registers are
// bounded (R 8: 72 and 18.5 us for 8191 tokens, 64 and 18.2; R 32: 194 without a bound).
template <typename T, int R>
__global__ void __launch_bounds__(kRouteWarps * 32, R <= 8 ? 8 : 4)
    route_kernel(const RouteParams r, const T* __restrict__ logits, long ld,
                 const float* __restrict__ bias, int tokens, int* __restrict__ selected,
                 float* __restrict__ weights, int vec) {
  __shared__ unsigned long long s_keys[kRouteWarps][32 * (R + 1)];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  void* shared = s_keys[threadIdx.x >> 5];
  const long t = (long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const T* row = logits + t * ld;
  float l[R];
  if (vec && lane * R + R <= r.experts) {
    load_logits<R>(row + lane * R, l);
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j)
      l[j] = lane * R + j < r.experts ? logit_at(row, lane * R + j) : -INFINITY;
  }
  // softmax: a NaN or +inf logit makes every score of the row NaN
  bool bad = false;
  if (r.softmax) {
#pragma unroll
    for (int j = 0; j < R; ++j) bad |= !(l[j] < INFINITY);
    bad = __any_sync(kFull, bad);
  }
  const bool by_logit = !bias && (r.top_groups == r.groups || r.group_top == 1) && !bad;
  float m = 0.0f, z = 1.0f;
  if (r.softmax) {
    m = l[0];
#pragma unroll
    for (int j = 1; j < R; ++j) m = fmaxf(m, l[j]);
    m = key_value(warp_max(order_key(m)));
    if (!by_logit || !r.renormalise) {  // else z divides out of the weights
      z = 0.0f;
#pragma unroll
      for (int j = 0; j < R; ++j) z += l[j] == -INFINITY ? 0.0f : expf(l[j] - m);
      z = bad ? __int_as_float(0x7fc00000) : warp_sum(z);
    }
  }
  int sel = 0;
  const bool sure = choose<R, float>(r, row, l, bias, by_logit, m, z, lane, shared, sel);
  if (!sure) {
    double zd = 1.0;
    if (r.softmax) {
      zd = 0.0;
#pragma unroll 1
      for (int e = lane; e < r.experts; e += 32) {
        const float v = logit_at(row, e);
        zd += v == -INFINITY ? 0.0 : exp((double)v - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) zd += __shfl_xor_sync(kFull, zd, o);
    }
    __syncwarp();
    if (!choose<R, double>(r, row, l, bias, false, m, zd, lane, shared, sel)) {
      __syncwarp();
      sel = choose_exact<R>(r, row, bias, m, zd, shared);
    }
  }
  // lane i: the weight of rank i
  float s = 0.0f, lv = 0.0f;
  if (lane < r.top_k) {
    lv = logit_at(row, sel);
    s = score(r, lv, m, z);
  }
  float w = s;
  if (r.renormalise) {
    const float sum = warp_sum(s);
    w = sum == 0.0f ? 0.0f : s / sum;
  }
  w *= r.scale;
  if (__any_sync(kFull, lane < r.top_k && s < 0x1p-100f && lv != -INFINITY))
    w = faint_weight(r, lv, m, z);
  if (lane < r.top_k) {
    selected[t * r.top_k + lane] = sel;
    weights[t * r.top_k + lane] = w;
  }
}

template <typename T>
cudaError_t route_t(const RouteParams& r, const T* logits, long ld, const float* bias, int tokens,
                    int* selected, float* weights, cudaStream_t st) {
  const dim3 grid((unsigned)((tokens + kRouteWarps - 1) / kRouteWarps)), block(kRouteWarps * 32);
  const int per = (r.experts + 31) / 32;
  const int vec = ld * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0;
  auto go = [&](auto kern) {
    return launch_pdl(kern, grid, block, 0, st, r, logits, ld, bias, tokens, selected, weights, vec);
  };
  if (per <= 1) return go(route_kernel<T, 1>);
  if (per <= 2) return go(route_kernel<T, 2>);
  if (per <= 4) return go(route_kernel<T, 4>);
  if (per <= 8) return go(route_kernel<T, 8>);
  if (per <= 16) return go(route_kernel<T, 16>);
  return go(route_kernel<T, 32>);
}

}  // namespace

cudaError_t launch_route(const RouteParams& r, bool bf16, const void* logits, long ld,
                         const float* bias, int tokens, int* selected, float* weights,
                         cudaStream_t st) {
  return bf16 ? route_t(r, static_cast<const __nv_bfloat16*>(logits), ld, bias, tokens, selected,
                        weights, st)
              : route_t(r, static_cast<const float*>(logits), ld, bias, tokens, selected, weights,
                        st);
}

}  // namespace lb
