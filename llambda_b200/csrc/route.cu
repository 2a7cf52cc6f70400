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
// (well under 1 in 10 tokens for logits of unit variance).
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

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

__device__ __forceinline__ float warp_max_value(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// The score of a logit; m is the largest logit and z the sum of exp(l - m)
// (softmax).  A row of -inf only scores 0.
template <typename F>
__device__ __forceinline__ F score(const RouteParams& r, float l, float m, F z) {
  if (l == -INFINITY) return F(0);
  return r.softmax ? exp_of((F)l - (F)m) / z : F(1) / (F(1) + exp_of(-(F)l));
}

// What the choice goes by.
template <typename F>
__device__ __forceinline__ F choice(const RouteParams& r, bool by_logit, const float* bias, float l,
                                    float m, F z, int e) {
  if (by_logit || l == -INFINITY) return (F)l;
  const F s = score<F>(r, l, m, z);
  return bias ? s + (F)__ldg(bias + e) : s;
}

// Bound on twice the error of an fp32 choice: the score's (expf, the division
// and, for softmax, the sum of exponentials: 4e-6 of the largest score smax in
// all) and the rounding of the sum with the bias.
__device__ __forceinline__ float choice_error(float c, float smax) {
  return 8e-6f * smax + 2.5e-7f * fabsf(c);
}

// The logit of expert e (the same on every lane), from the lane that holds it.
template <int R>
__device__ __forceinline__ float expert_logit(const float (&l)[R], int e) {
  float v = l[0];
#pragma unroll
  for (int j = 1; j < R; ++j)
    if (j == e >> 5) v = l[j];
  return __shfl_sync(kFull, v, e & 31);
}

// The choice of one token by one warp: lane L holds experts L, L + 32, ....
// Rank i's expert goes to lane i.  F = float: returns false when some deciding
// comparison was too close (by_logit: the compared values are exact).
template <int R, typename F>
__device__ __forceinline__ bool choose(const RouteParams& r, const float (&l)[R], const float* bias,
                                       bool by_logit, float m, F z, int lane, int& sel) {
  using K = decltype(order_key(F(0)));
  const bool check = sizeof(F) == 4 && !by_logit;
  K key[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = j * 32 + lane;
    key[j] = e < r.experts ? order_key(choice<F>(r, by_logit, bias, l[j], m, z, e)) : K(0);
  }
  bool sure = true;
  const float smax = r.softmax ? 1.0f / (float)z : 1.0f;
  if (r.top_groups < r.groups) {
    const int size = r.experts / r.groups;
    K gkey = 0;  // lane g: group g's score
    for (int g = 0; g < r.groups; ++g) {
      const int lo = g * size, hi = lo + size;
      K a = 0, b = 0;  // this lane's two largest
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int e = j * 32 + lane;
        const K v = e >= lo && e < hi ? key[j] : K(0);
        b = max(b, min(a, v));
        a = max(a, v);
      }
      K best = warp_max(a);
      if (r.group_top == 2) {
        const unsigned owner = __ballot_sync(kFull, a == best);
        const K second = warp_max(lane == __ffs(owner) - 1 ? b : a);
        best = order_key(key_value(best) + key_value(second));
      }
      if (lane == g) gkey = best;
    }
    unsigned kept = 0;
    K last = 0;
    for (int i = 0; i < r.top_groups; ++i) {
      last = warp_max(gkey);
      const int g = __ffs(__ballot_sync(kFull, gkey == last)) - 1;
      kept |= 1u << g;
      if (lane == g) gkey = 0;
    }
    if (check) {
      // the best group left out against the worst one kept (a NaN compares false)
      const F in = key_value(last), out = key_value(warp_max(gkey));
      if (in - out <= F(2) * (F)choice_error((float)in, smax)) sure = false;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int e = j * 32 + lane;
      if (e < r.experts && !(kept >> (e / size) & 1u)) key[j] = 0;
    }
  }
  K prev = 0;
  int prev_e = 0;
  for (int i = 0; i <= r.top_k; ++i) {
    if (i == r.top_k && !check) break;
    K a = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (key[j] > a) a = key[j], at = j;
    const K best = warp_max(a);
    if (best == 0) break;  // no expert left to compare with
    const int e = __reduce_min_sync(kFull, a == best ? at * 32 + lane : 0x7fffffff);
    if (i < r.top_k && lane == i) sel = e;
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (e == j * 32 + lane) key[j] = 0;
    if (check && i > 0) {
      const F c = key_value(prev), d = key_value(best);
      // equal logits and biases are a true tie, which the index decides
      if (c - d <= (F)choice_error((float)c, smax) &&
          !(expert_logit(l, prev_e) == expert_logit(l, e) && bias &&
            __ldg(bias + prev_e) == __ldg(bias + e)))
        sure = false;
    }
    prev = best;
    prev_e = e;
  }
  return sure;
}

__device__ __forceinline__ float logit_at(const float* p, long i) { return __ldg(p + i); }
__device__ __forceinline__ float logit_at(const __nv_bfloat16* p, long i) {
  return __bfloat162float(p[i]);
}

template <typename T, int R>
__global__ void __launch_bounds__(kRouteWarps * 32)
    route_kernel(const RouteParams r, const T* __restrict__ logits, long ld,
                 const float* __restrict__ bias, int tokens, int* __restrict__ selected,
                 float* __restrict__ weights) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  const long t = (long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const T* row = logits + t * ld;
  float l[R];
  bool nan = false;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = j * 32 + lane;
    l[j] = e < r.experts ? logit_at(row, e) : -INFINITY;
    nan |= isnan(l[j]);
  }
  float m = 0.0f, z = 1.0f;
  if (r.softmax) {
    m = l[0];
#pragma unroll
    for (int j = 1; j < R; ++j) m = fmaxf(m, l[j]);
    m = warp_max_value(m);
    z = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j) z += l[j] == -INFINITY ? 0.0f : expf(l[j] - m);
    z = warp_sum(z);
    nan = isnan(z);  // a NaN or +inf logit makes every score NaN
  }
  const bool scores_order =
      !bias && (r.top_groups == r.groups || r.group_top == 1) && !(r.softmax && nan);
  int sel = 0;
  if (!choose<R, float>(r, l, bias, scores_order, m, z, lane, sel)) {
    double zd = 1.0;
    if (r.softmax) {
      zd = 0.0;
#pragma unroll 1
      for (int j = 0; j < R; ++j) {
        const int e = j * 32 + lane;
        const float v = e < r.experts ? logit_at(row, e) : -INFINITY;
        zd += v == -INFINITY ? 0.0 : exp((double)v - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) zd += __shfl_xor_sync(kFull, zd, o);
    }
    choose<R, double>(r, l, bias, false, m, zd, lane, sel);
  }
  // lane i: the weight of rank i
  float s = 0.0f;
  if (lane < r.top_k) s = score<float>(r, logit_at(row, sel), m, z);
  float w = s;
  if (r.renormalise) {
    const float sum = warp_sum(s);
    w = sum == 0.0f ? 0.0f : s / sum;
  }
  if (lane < r.top_k) {
    selected[t * r.top_k + lane] = sel;
    weights[t * r.top_k + lane] = w * r.scale;
  }
}

template <typename T>
cudaError_t route_t(const RouteParams& r, const T* logits, long ld, const float* bias, int tokens,
                    int* selected, float* weights, cudaStream_t st) {
  const dim3 grid((unsigned)((tokens + kRouteWarps - 1) / kRouteWarps)), block(kRouteWarps * 32);
  const int per = (r.experts + 31) / 32;
  auto go = [&](auto kern) {
    return launch_pdl(kern, grid, block, 0, st, r, logits, ld, bias, tokens, selected, weights);
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
