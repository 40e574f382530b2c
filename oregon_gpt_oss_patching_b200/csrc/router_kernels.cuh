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
// One warp serves one token.  A lane holds up to 8 experts (whole lanes to a group) as keys: the upper 24 bits of the value in
// an order of unsigned integers, and 255 - expert below, so that keys differ and the larger one is the one to elect.  The lane
// sorts its keys; a round of the election is one warp-wide integer maximum (`redux.sync`) of the lanes' first keys, and the lane
// that has it moves up its list.  Instructions bound the kernel, not memory (a few MB): 32771 tokens, 8 of 256 experts, sigmoid,
// bias, 4 of 8 groups take @FWD@ us forward and @BWD@ us backward.  (Full keys with two maxima a round, unsorted lists and groups
// summed through shared memory, as the slow path below has it: 89 us.)
//
// 24 bits hold every bf16 and fp16 logit, so the choice is exact where neither bias nor groups take part (scores rise with
// logits).  Otherwise lane j looks at the gap between the (j - 1)-th and the j-th value elected, one more than is wanted among
// them, and at the border between groups.  Where a gap is not wider than what the keys and fp32 lose (and the two do not come
// from the same logit and bias, where the lower index is right), the warp elects again, in full fp32 and, where that cannot tell
// either, in fp64: about one token in 300 of random ones.
#pragma once
#include <math_constants.h>

#include "elem_types.cuh"

namespace b200moe {

using b200train::Elem;
using b200train::pack;
using b200train::unpack;

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
  int vector;               // a lane's experts can be loaded at once
  int slow;                 // top_k or the groups are beyond the quick election
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

// The election in full precision, for any groups and top_k: lane j's return is the j-th expert.  `row` is shared memory of this warp.
template <typename T, int VPL>
__device__ __noinline__ int elect_slowly(const RouterArgs& a, const T* logits, int lane, double* row) {
  float l[VPL], b[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    l[i] = e < a.experts ? Elem<T>::load1(logits + e) : -CUDART_INF_F;
    b[i] = a.bias != nullptr && e < a.experts ? a.bias[e] : 0.f;
  }
  bool close;
  if (a.bias == nullptr && a.groups == 1) return elect<float, VPL, false>(l, b, a, lane, nullptr, false, close).expert;
  const int e = elect<float, VPL, true>(l, b, a, lane, reinterpret_cast<float*>(row), true, close).expert;
  if (!close) return e;   // (the same in every lane)
  return elect<double, VPL, true>(l, b, a, lane, row, false, close).expert;
}

constexpr float kKeyStep = 2.f / 32768.f;   // two steps of a key's 15 bits of mantissa, relative
constexpr float kValueError = 4e-6f;        // of two values of 1 + |v|, with their scores' errors

__device__ __forceinline__ uint32_t make_key(float v, int expert) { return (order_key(v) & 0xffffff00u) | (255u - expert); }
// the middle of the values that share a key's upper 24 bits; -inf for a masked expert's
__device__ __forceinline__ float key_value(uint32_t key) {
  if (key <= 0x007fffffu) return -CUDART_INF_F;
  const uint32_t u = (key & 0xffffff00u) | 0x80u;
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ void sort_pair(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}
// falling order (Batcher's odd-even merge)
template <int VPL>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[VPL]) {
  if constexpr (VPL >= 2) {
#pragma unroll
    for (int i = 0; i < VPL; i += 2) sort_pair(k[i], k[i + 1]);
  }
  if constexpr (VPL >= 4) {
#pragma unroll
    for (int i = 0; i < VPL; i += 4) {
      sort_pair(k[i], k[i + 2]);
      sort_pair(k[i + 1], k[i + 3]);
      sort_pair(k[i + 1], k[i + 2]);
    }
  }
  if constexpr (VPL == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sort_pair(k[i], k[i + 4]);
    sort_pair(k[2], k[4]);
    sort_pair(k[3], k[5]);
    sort_pair(k[1], k[2]);
    sort_pair(k[3], k[4]);
    sort_pair(k[5], k[6]);
  }
}

// `VPL` neighbouring elements from p on, `n` of which exist; in one or two loads where they lie on a grid of their own size.
template <typename T, int VPL>
__device__ __forceinline__ void load_run(const T* p, int n, bool vector, float (&l)[VPL]) {
  if (vector) {
    constexpr int kBytes = VPL * (int)sizeof(T);
    if constexpr (kBytes == 32) {
      unpack<T>(*reinterpret_cast<const uint4*>(p), l);
      unpack<T>(*reinterpret_cast<const uint4*>(p + VPL / 2), l + VPL / 2);
    } else if constexpr (kBytes == 16) {
      unpack<T>(*reinterpret_cast<const uint4*>(p), l);
    } else {
      struct alignas(kBytes) Run {
        T v[VPL];
      };
      const Run run = *reinterpret_cast<const Run*>(p);
#pragma unroll
      for (int i = 0; i < VPL; ++i) l[i] = Elem<T>::load1(&run.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) l[i] = i < n ? Elem<T>::load1(p + i) : -CUDART_INF_F;
  }
}

template <typename T, int VPL>
__device__ __forceinline__ void store_run(T* p, int n, bool vector, const float (&g)[VPL]) {
  if (vector) {
    constexpr int kBytes = VPL * (int)sizeof(T);
    if constexpr (kBytes == 32) {
      *reinterpret_cast<uint4*>(p) = pack<T>(g);
      *reinterpret_cast<uint4*>(p + VPL / 2) = pack<T>(g + VPL / 2);
    } else if constexpr (kBytes == 16) {
      *reinterpret_cast<uint4*>(p) = pack<T>(g);
    } else {
      struct alignas(kBytes) Run {
        T v[VPL];
      };
      Run run;
#pragma unroll
      for (int i = 0; i < VPL; ++i) Elem<T>::store1(&run.v[i], g[i]);
      *reinterpret_cast<Run*>(p) = run;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i < n) Elem<T>::store1(p + i, g[i]);
  }
}

// A score fit to be elected by: expf and a true quotient cost three times as much and tell no more apart.
__device__ __forceinline__ float quick_sigmoid(float l) { return __fdividef(1.f, 1.f + __expf(-l)); }

// kValues: a bias or groups take part.  The host sees to it that a group has whole lanes (their number a power of two) and
// top_k < 32, or asks for the slow path at once.
template <typename T, int VPL, bool kValues>
__global__ void __launch_bounds__(kRouterThreads) router_topk_kernel(const __grid_constant__ RouterArgs a) {
  constexpr bool kExact = !kValues && sizeof(T) == 2;
  __shared__ double rows[kValues ? kRouterThreads / 32 : 1][kValues ? 32 * VPL : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x * (kRouterThreads / 32) + warp;
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  float l[VPL], m = 0.f, z = 1.f;
  uint32_t key[VPL];
  const int groups = a.slow ? 1 : a.groups, part = 32 / groups, size = a.experts / groups, per = (size + part - 1) / part;   // lanes a group, experts a group, a lane
  const int group = lane / part, place = lane % part * per;
  const int first = group * size + place, mine = max(0, min(per, size - place));
  load_run<T, VPL>(row + first, mine, a.vector != 0, l);
  if (!a.sigmoid && (kValues || !a.renormalize)) {   // the softmax's maximum and sum
    m = l[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = l[i] > m || l[i] != l[i] ? l[i] : m;
    m = warp_max(m);
    z = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) z += l[i] == -CUDART_INF_F ? 0.f : expf(l[i] - m);
    z = warp_add(z);
  }
  auto value = [&](float x, int e) -> float {
    if (!kValues) return x;
    if (x == -CUDART_INF_F) return x;
    const float s = a.sigmoid ? quick_sigmoid(x) : __fdividef(expf(x - m), z);
    return a.bias != nullptr ? s + a.bias[e] : s;
  };
  uint32_t won = 0;   // lane j's: the j-th key
  bool sure = !a.slow;
  if (sure) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = i < mine ? make_key(value(l[i], first + i), first + i) : 0u;
    sort_keys<VPL>(key);
    if (kValues && a.groups > 1) {
      float best = key_value(key[0]), next = VPL > 1 ? key_value(key[VPL > 1 ? 1 : 0]) : -CUDART_INF_F;
      for (int o = part >> 1; o > 0; o >>= 1) {
        const float f = __shfl_xor_sync(0xffffffffu, best, o), s = __shfl_xor_sync(0xffffffffu, next, o);
        next = fmaxf(fminf(best, f), fmaxf(next, s));
        best = fmaxf(best, f);
      }
      const float sum = next == -CUDART_INF_F ? best : best + next;
      const float slack = best == -CUDART_INF_F ? 0.f : kKeyStep * (fabsf(best) + (next == -CUDART_INF_F ? 0.f : fabsf(next))) + 2.f * kValueError;
      int ahead = 0;
      for (int g = 0; g < a.groups; ++g) {
        const float other = __shfl_sync(0xffffffffu, sum, g * part);
        ahead += other > sum || (other == sum && g < group);
      }
      const bool open = ahead < a.top_groups;
      // the narrowest of the gaps between an open group and a closed one
      if (a.top_groups < a.groups) {
        const float in = warp_max(open ? -sum : -CUDART_INF_F), out = warp_max(open ? -CUDART_INF_F : sum);
        const float most = warp_max(slack);
        sure = -in - out > 2.f * most || (-in == -CUDART_INF_F && out == -CUDART_INF_F);
        sure = sure && key[0] < 0xffffff00u;   // (no NaN)
        sure = __all_sync(0xffffffffu, sure);
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i) key[i] = open ? key[i] : 0u;
    }
    const int rounds = kExact ? a.top_k : a.top_k + 1;
    for (int j = 0; j < rounds; ++j) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
      if (lane == j) won = top;
      const bool pop = key[0] == top;
#pragma unroll
      for (int i = 0; i + 1 < VPL; ++i) key[i] = pop ? key[i + 1] : key[i];
      key[VPL - 1] = pop ? 0u : key[VPL - 1];
    }
  }
  int expert = 255 - (int)(won & 255u);
  const bool chosen = lane < a.top_k;
  float x = -CUDART_INF_F;
  if (!a.slow && (chosen || (!kExact && lane == a.top_k && won != 0u))) x = Elem<T>::load1(row + expert);
  if (!kExact) {
    if (!a.slow) {
      float b = 0.f, v = x;
      if (kValues && lane <= a.top_k && won != 0u) {
        v = value(x, expert);
        b = a.bias != nullptr ? a.bias[expert] : 0.f;
      }
      const float pv = __shfl_up_sync(0xffffffffu, v, 1), px = __shfl_up_sync(0xffffffffu, x, 1), pb = __shfl_up_sync(0xffffffffu, b, 1);
      const bool masked = x == -CUDART_INF_F && px == -CUDART_INF_F;
      const float gap = pv - v, error = kValues ? kValueError * (1.f + fabsf(v)) : 0.f;
      bool fine = true;
      if (lane > 0 && lane < a.top_k) fine = masked || (px == x && pb == b) || gap > error;
      else if (lane == a.top_k) fine = won == 0u || masked || gap > error + kKeyStep * fabsf(pv);
      sure = __all_sync(0xffffffffu, fine) && sure;
    }
    if (!sure) {   // (the same in every lane)
      expert = elect_slowly<T, VPL>(a, row, lane, rows[kValues ? warp : 0]);
      x = chosen ? Elem<T>::load1(row + expert) : -CUDART_INF_F;
    }
  }
  // the weights of the elected
  float s;
  if (a.sigmoid) {
    s = chosen ? 1.f / (1.f + expf(-x)) : 0.f;
  } else {
    if (a.renormalize) m = warp_max(chosen ? x : -CUDART_INF_F);
    s = chosen && x != -CUDART_INF_F ? expf(x - m) : 0.f;
    if (!a.renormalize) s = z == 0.f ? 0.f : s / z;
  }
  if (a.renormalize) {
    const float sum = warp_add(s);
    s = sum == 0.f ? 0.f : s / sum;
  }
  if (chosen) {
    Elem<T>::store1(static_cast<T*>(a.weights) + (long long)t * a.top_k + lane, s * a.scale);
    a.indices[(long long)t * a.top_k + lane] = expert;
  }
}

struct RouterBwdArgs {
  const void* logits;
  long long stride;
  const long long* indices;   // (tokens, top_k)
  const void* dweights;       // (tokens, top_k)
  void* dlogits;              // (tokens, experts) contiguous
  int tokens, experts, top_k, sigmoid, renormalize;
  int vector_in, vector_out;   // a lane's experts can be loaded, stored at once
  float scale;
};

// With d_j = scale * dw_j and, renormalised, r_j = s_j / sum_S s and d_j <- (d_j - sum_S d r) / sum_S s:
//   sigmoid   dl_j = d_j s_j (1 - s_j) for the chosen, 0 elsewhere
//   softmax   dl_i = s_i (d_i - sum_S d s), d_i = 0 where i is not chosen; renormalised that is r_j (d_j - sum_S d r), 0 elsewhere
template <typename T, int VPL>
__global__ void __launch_bounds__(kRouterThreads) router_topk_bwd_kernel(const __grid_constant__ RouterBwdArgs a) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * (kRouterThreads / 32) + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  T* out = static_cast<T*>(a.dlogits) + (long long)t * a.experts;
  int e = -1;
  float lj = -CUDART_INF_F, d = 0.f;
  if (lane < a.top_k) {
    const long long index = a.indices[(long long)t * a.top_k + lane];
    e = index >= 0 && index < a.experts ? (int)index : -1;
    if (e >= 0) lj = Elem<T>::load1(row + e);
    d = Elem<T>::load1(static_cast<const T*>(a.dweights) + (long long)t * a.top_k + lane) * a.scale;
  }
  float g[VPL], chosen;   // the gradients of a run of experts of this lane's; of lane j's chosen expert
#pragma unroll
  for (int i = 0; i < VPL; ++i) g[i] = 0.f;
  const int first = lane * VPL, n = max(0, min(VPL, a.experts - first));
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
    float l[VPL], z = 0.f;
    load_run<T, VPL>(row + first, n, a.vector_in != 0 && n == VPL, l);
    float m = l[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = l[i] > m || l[i] != l[i] ? l[i] : m;
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
  // the whole row first, then the chosen experts over it (stores of one warp in this order)
  store_run<T, VPL>(out + first, n, a.vector_out != 0 && n == VPL, g);
  __syncwarp();
  if (e >= 0) Elem<T>::store1(out + e, chosen);
}

}  // namespace b200moe
