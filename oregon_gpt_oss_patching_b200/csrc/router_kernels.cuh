// Routing of tokens to experts: scores, a bias for the choice, groups, the best top_k and their weights, and the gradient.
//
//   s = softmax(l) or sigmoid(l);   v = s + bias   (a logit of -inf: s = 0 and v = -inf, whatever the bias)
//   groups: a group's value is the sum of its two largest v that are not -inf (-inf where there is none); the experts of the
//           top_groups best groups stand for election
//   S = the top_k largest v, ties to the lowest index;   w_j = scale * s_j / (sum_S s if renormalize else 1), 0 where that sum is 0
//
// GptOssTopKRouter.forward (transformers/models/gpt_oss/modeling_gpt_oss.py:126-133) is softmax, no bias, no groups, renormalised:
// the softmax over the chosen logits.
//
// One warp serves one token: lane L holds the experts L, L + 32, ... in registers; a round of the election is two
// warp-wide integer reductions (`redux.sync`), the largest key and the lowest expert that has it.
//
// Where neither bias nor groups take part the keys are the logits themselves (scores rise with logits), and the choice is
// exact.  Otherwise it goes by values, which fp32 gets wrong by a few 2^-24: the warp elects by fp32 values and looks at the
// gaps between neighbours of the ranking and at the border between groups; where one is too small to be trusted (and the
// two do not come from the same logit and bias, where the lower index is right), it elects again with values in fp64.
#pragma once
#include <math_constants.h>

#include "elem_types.cuh"

namespace b200moe {

using b200train::Elem;

constexpr int kRouterThreads = 256;
constexpr int kRouterMaxExperts = 256;   // 8 a lane
constexpr int kRouterMaxTopK = 32;       // one a lane
constexpr int kRouterMaxGroups = 32;     // one lane a group at least

// fp32 and fp64 values as unsigned keys in the same order; NaN above everything (as torch.topk has it), -0 as 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  if (v != v) return 0xffffffffu;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  if (v != v) return ~0ull;
  return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  return k;
}
template <typename V>
__device__ __forceinline__ V warp_max(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const V other = __shfl_xor_sync(0xffffffffu, v, o);
    v = other > v || other != other ? other : v;   // (a NaN wins)
  }
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_add(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

struct RouterArgs {
  const void* logits;       // (tokens, experts), row stride below
  long long stride;
  const float* bias;        // (experts) or nullptr
  void* weights;            // (tokens, top_k)
  long long* indices;       // (tokens, top_k)
  int tokens, experts, top_k, groups, top_groups;
  int sigmoid, renormalize;
  float scale;
};

// The scores of this lane's experts, in V's precision.
template <typename V, int VPL>
__device__ __forceinline__ void scores_of(const float (&l)[VPL], bool sigmoid, V (&s)[VPL]) {
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) s[i] = V(1) / (V(1) + exp_of(-V(l[i])));
  } else {
    float m = l[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = l[i] > m || l[i] != l[i] ? l[i] : m;
    m = warp_max(m);
    V z = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      s[i] = l[i] == -CUDART_INF_F ? V(0) : exp_of(V(l[i]) - V(m));
      z += s[i];
    }
    z = warp_add(z);
#pragma unroll
    for (int i = 0; i < VPL; ++i) s[i] = z == V(0) ? V(0) : s[i] / z;
  }
}

template <typename V>
struct Top2 {
  V first, second;
  __device__ __forceinline__ void add(V v) {
    if (v > first || v != v) { second = first; first = v; }
    else if (v > second) second = v;
  }
  __device__ __forceinline__ V sum() const { return second > V(-CUDART_INF_F) ? first + second : first; }
};

// Which groups stand for election, as a bit mask.  `row` (shared, of this warp) holds the values by expert.  The lanes are
// shared out: `part` of them (a power of two) walk one group.  `close` is set where the border between the groups chosen
// and those left is narrower than `margin` (times 1 + the value).
template <typename V>
__device__ __forceinline__ uint32_t open_groups(const V* row, const RouterArgs& a, int lane, V margin, bool& close) {
  int part = 32;
  while (part * a.groups > 32) part >>= 1;
  const int size = a.experts / a.groups, g = lane / part, p = lane % part;
  Top2<V> best{V(-CUDART_INF_F), V(-CUDART_INF_F)};
  if (g < a.groups)
    for (int j = p; j < size; j += part) best.add(row[g * size + j]);
  for (int o = part >> 1; o > 0; o >>= 1) {
    const V f = __shfl_xor_sync(0xffffffffu, best.first, o), s = __shfl_xor_sync(0xffffffffu, best.second, o);
    best.add(f);
    best.add(s);
  }
  // lane g now ranks group g among all
  const V sums = best.sum();
  const V mine = __shfl_sync(0xffffffffu, sums, (lane * part) & 31);
  const auto key = order_key(mine);
  int ahead = 0;
  for (int other = 0; other < a.groups; ++other) {
    const auto k = __shfl_sync(0xffffffffu, key, other);
    ahead += k > key || (k == key && other < lane);
  }
  const bool chosen = lane < a.groups && ahead < a.top_groups;
  const uint32_t mask = __ballot_sync(0xffffffffu, chosen);
  if (margin > V(0) && a.top_groups < a.groups) {
    const uint32_t last_in = __ballot_sync(0xffffffffu, lane < a.groups && ahead == a.top_groups - 1);
    const uint32_t first_out = __ballot_sync(0xffffffffu, lane < a.groups && ahead == a.top_groups);
    const V in = __shfl_sync(0xffffffffu, mine, __ffs(last_in) - 1), out = __shfl_sync(0xffffffffu, mine, __ffs(first_out) - 1);
    // (two groups without an expert that is not masked are a true tie)
    close = !(in - out > margin * (V(1) + fabs(in))) && !(in == V(-CUDART_INF_F) && out == V(-CUDART_INF_F));
  }
  return mask;
}

// An election's outcome: lane j (< top_k) holds the j-th expert and its logit.
struct Elected {
  int expert;
  float logit;
};

// V: float or double values (kValues), or the logits themselves (!kValues).
template <typename V, int VPL, bool kValues>
__device__ __forceinline__ Elected elect(const float (&l)[VPL], const float (&b)[VPL], const RouterArgs& a, int lane, V* row, bool check, bool& close) {
  using Key = decltype(order_key(V(0)));
  Key key[VPL];
  close = false;
  if constexpr (kValues) {
    V v[VPL];
    scores_of<V, VPL>(l, a.sigmoid != 0, v);
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = l[i] == -CUDART_INF_F ? V(-CUDART_INF_F) : v[i] + V(b[i]);
    uint32_t open = 0xffffffffu;
    if (a.groups > 1) {
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (lane + 32 * i < a.experts) row[lane + 32 * i] = v[i];
      __syncwarp();
      open = open_groups<V>(row, a, lane, check ? V(8e-6) : V(0), close);
      __syncwarp();
    }
    const int size = a.experts / a.groups;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      key[i] = e < a.experts && (a.groups == 1 || (open >> (e / size)) & 1u) ? order_key(v[i]) : Key(0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = lane + 32 * i < a.experts ? order_key(V(l[i])) : Key(0);
  }
  Elected out{0, 0.f};
  float last_l = 0.f, last_b = 0.f;
  V last_v = 0;
  // one round more than is elected, to see the gap behind the last one
  const int rounds = kValues && check && a.top_k < a.experts ? a.top_k + 1 : a.top_k;
  for (int j = 0; j < rounds; ++j) {
    Key best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < VPL; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
    const Key top = warp_max_key(best);
    if (kValues && top == Key(0)) break;   // (no expert is left behind the last one elected)
    const int e = (int)__reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
    const int slot = e >> 5, owner = e & 31;
    float le = 0.f, be = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i == slot) {
        le = l[i];
        be = b[i];
        if (lane == owner) key[i] = Key(0);
      }
    le = __shfl_sync(0xffffffffu, le, owner);
    if constexpr (kValues) {
      if (check) {
        be = __shfl_sync(0xffffffffu, be, owner);
        // the value back from its key
        const uint32_t bits = (top & 0x80000000u) ? (uint32_t)top & 0x7fffffffu : ~(uint32_t)top;
        const V v = V(__uint_as_float(bits));
        const bool same = __float_as_uint(le) == __float_as_uint(last_l) && (be == last_b || le == -CUDART_INF_F);
        if (j > 0 && !same && !(last_v - v > V(4e-6) * (V(1) + fabs(v)))) close = true;
        last_l = le;
        last_b = be;
        last_v = v;
      }
    }
    if (lane == j) out = Elected{e, le};
  }
  return out;
}

template <typename T, int VPL, bool kValues>
__global__ void __launch_bounds__(kRouterThreads) router_topk_kernel(const RouterArgs a) {
  __shared__ double rows[kValues ? kRouterThreads / 32 : 1][kValues ? 32 * VPL : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x * (kRouterThreads / 32) + warp;
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  float l[VPL], b[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    l[i] = e < a.experts ? Elem<T>::load1(row + e) : -CUDART_INF_F;
    b[i] = kValues && a.bias != nullptr && e < a.experts ? a.bias[e] : 0.f;
  }
  bool close = false;
  Elected w = elect<float, VPL, kValues>(l, b, a, lane, reinterpret_cast<float*>(rows[kValues ? warp : 0]), kValues, close);
  if constexpr (kValues) {
    if (close) {   // (the same in every lane)
      bool ignored;
      w = elect<double, VPL, true>(l, b, a, lane, rows[warp], false, ignored);
    }
  }
  // the weights of the elected, lane j's being the j-th
  const bool mine = lane < a.top_k;
  float s;
  if (a.sigmoid) {
    s = mine ? 1.f / (1.f + expf(-w.logit)) : 0.f;
  } else {
    float m;
    if (a.renormalize) {
      m = warp_max(mine ? w.logit : -CUDART_INF_F);
    } else {
      m = l[0];
#pragma unroll
      for (int i = 1; i < VPL; ++i) m = l[i] > m || l[i] != l[i] ? l[i] : m;
      m = warp_max(m);
    }
    s = mine && w.logit != -CUDART_INF_F ? expf(w.logit - m) : 0.f;
    if (!a.renormalize) {
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) z += l[i] == -CUDART_INF_F ? 0.f : expf(l[i] - m);
      z = warp_add(z);
      s = z == 0.f ? 0.f : s / z;
    }
  }
  if (a.renormalize) {
    const float sum = warp_add(s);
    s = sum == 0.f ? 0.f : s / sum;
  }
  if (mine) {
    Elem<T>::store1(static_cast<T*>(a.weights) + (long long)t * a.top_k + lane, s * a.scale);
    a.indices[(long long)t * a.top_k + lane] = w.expert;
  }
}

struct RouterBwdArgs {
  const void* logits;
  long long stride;
  const long long* indices;   // (tokens, top_k)
  const void* dweights;       // (tokens, top_k)
  void* dlogits;              // (tokens, experts) contiguous
  int tokens, experts, top_k, sigmoid, renormalize;
  float scale;
};

// With d_j = scale * dw_j and, renormalised, r_j = s_j / sum_S s and d_j <- (d_j - sum_S d r) / sum_S s:
//   sigmoid   dl_j = d_j s_j (1 - s_j) for the chosen, 0 elsewhere
//   softmax   dl_i = s_i (d_i - sum_S d s), d_i = 0 where i is not chosen; renormalised that is r_j (d_j - sum_S d r), 0 elsewhere
template <typename T, int VPL>
__global__ void __launch_bounds__(kRouterThreads) router_topk_bwd_kernel(const RouterBwdArgs a) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * (kRouterThreads / 32) + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  const bool mine = lane < a.top_k;
  int e = -1;
  float lj = -CUDART_INF_F, d = 0.f;
  if (mine) {
    const long long index = a.indices[(long long)t * a.top_k + lane];
    e = index >= 0 && index < a.experts ? (int)index : -1;
    if (e >= 0) lj = Elem<T>::load1(row + e);
    d = Elem<T>::load1(static_cast<const T*>(a.dweights) + (long long)t * a.top_k + lane) * a.scale;
  }
  float g[VPL], chosen;   // this lane's experts' gradients; lane j's chosen expert's
#pragma unroll
  for (int i = 0; i < VPL; ++i) g[i] = 0.f;
  if (a.sigmoid) {
    const float x = expf(-fabsf(lj)), s = (lj >= 0.f ? 1.f : x) / (1.f + x);   // (no overflow on either side)
    const float slope = x / ((1.f + x) * (1.f + x));
    if (a.renormalize) {
      const float sum = warp_add(e >= 0 ? s : 0.f);
      const float dot = warp_add(e >= 0 ? d * s : 0.f);
      d = sum == 0.f ? 0.f : (d - dot / sum) / sum;
    }
    chosen = d * slope;
  } else if (a.renormalize) {
    const float m = warp_max(lj);
    const float s = lj == -CUDART_INF_F ? 0.f : expf(lj - m);
    const float sum = warp_add(s);
    const float r = sum == 0.f ? 0.f : s / sum;
    chosen = r * (d - warp_add(e >= 0 ? d * r : 0.f));
  } else {
    float l[VPL], m = -CUDART_INF_F, z = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      l[i] = lane + 32 * i < a.experts ? Elem<T>::load1(row + lane + 32 * i) : -CUDART_INF_F;
      m = l[i] > m || l[i] != l[i] ? l[i] : m;
    }
    m = warp_max(m);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      g[i] = l[i] == -CUDART_INF_F ? 0.f : expf(l[i] - m);
      z += g[i];
    }
    z = warp_add(z);
    const float s = lj == -CUDART_INF_F || z == 0.f ? 0.f : expf(lj - m) / z;
    const float dot = warp_add(e >= 0 ? d * s : 0.f);
    chosen = s * (d - dot);
#pragma unroll
    for (int i = 0; i < VPL; ++i) g[i] = z == 0.f ? 0.f : -(g[i] / z) * dot;
  }
  for (int j = 0; j < a.top_k; ++j) {
    const int ej = __shfl_sync(0xffffffffu, e, j);
    const float cj = __shfl_sync(0xffffffffu, chosen, j);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (ej == lane + 32 * i) g[i] = cj;
  }
  T* out = static_cast<T*>(a.dlogits) + (long long)t * a.experts;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (lane + 32 * i < a.experts) Elem<T>::store1(out + lane + 32 * i, g[i]);
}

}  // namespace b200moe
