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
// The quick election (top_k <= 8; 1, 2, 4 or 8 groups): 8 lanes serve a token, 4 tokens a warp.  A lane turns its up to 32
// experts (whole lanes to a group) into keys: the upper 24 bits of the value in an order of unsigned integers, and 255 - expert
// below, so that keys differ and the larger one is the one to elect.  It sorts them by eights with a network, keeps the best 8
// (or 4, where top_k allows), and three exchanges between the lanes leave the token's best in all of them.  Instructions bound
// the kernel, not memory (a few MB): 32771 tokens, 8 of 256 experts, sigmoid, bias, 4 of 8 groups take 38 us forward (26 us
// without the doubtful tokens, below), on logits alone 12.5 us, and 8 us backward.  (A warp a token with a warp-wide maximum a
// round: 66, 25 and 12 us; that with full keys, two maxima a round and groups summed through shared memory: 89 and 37 us.)
//
// 24 bits hold every bf16 and fp16 logit, so the order is exact where no bias takes part (scores rise with logits).  Otherwise a lane looks at the gap between its and the last lane's value, at the one behind the last elected and at
// the border between groups.  Where a gap is not wider than what the keys and fp32 lose (and the two do not come from the
// same logit and bias, where the lower index is right), the whole warp elects for that token again, in fp64: about one token
// in 450 of random ones.
#pragma once
#include <math_constants.h>

#include "elem_types.cuh"

namespace b200moe {

using b200train::Elem;
using b200train::pack;
using b200train::unpack;

constexpr int kRouterThreads = 256;
constexpr int kRouterMaxExperts = 256;   // 8 a lane of the slow election, 32 a lane of the quick one
constexpr int kRouterMaxTopK = 32;       // one a lane
constexpr int kRouterMaxGroups = 32;     // one lane a group at least
constexpr int kQuickLanes = 8;           // of a token
constexpr int kQuickTokens = kRouterThreads / kQuickLanes;

// fp32 and fp64 values as unsigned keys in the same order; NaN above everything (as torch.topk has it), -0 as 0.  (An fp32 sum makes
// 0 of -0 and the one positive NaN, 0x7fffffff, of any.)
__device__ __forceinline__ uint32_t order_key(float v) {
  const int b = __float_as_int(v + 0.f);
  return (uint32_t)(b ^ (b >> 31 | (int)0x80000000));
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  if (v != v) return ~0ull;
  return (b >> 63) ? ~b : b | (1ull << 63);
}

// Sums and maxima over runs of `width` lanes (a power of two).
template <typename V>
__device__ __forceinline__ V lanes_add(V v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V lanes_max(V v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) {
    const V other = __shfl_xor_sync(0xffffffffu, v, o);
    v = other > v || other != other ? other : v;   // (a NaN wins)
  }
  return v;
}

struct RouterArgs {
  const void* logits;       // (tokens, experts), row stride below
  long long stride;
  const float* bias;        // (experts) or nullptr
  void* weights;            // (tokens, top_k)
  long long* indices;       // (tokens, top_k)
  int tokens, experts, top_k, groups, top_groups;
  int sigmoid, renormalize;
  int vector, vector_bias;  // a lane's experts, their biases can be loaded at once
  float scale;
};

// The value of a key.
__device__ __forceinline__ double value_of(unsigned long long key) {
  return __longlong_as_double((long long)((key >> 63) ? key & ~(1ull << 63) : ~key));
}

// The slow election: any groups and top_k, values in fp64, a whole warp a token; lane j's return is the j-th expert.  `row` (shared,
// of this warp) holds the values' keys by expert, 0 where an expert cannot be elected any more.  One token waits for it, so
// latency counts: no branch keeps neighbouring experts' exponentials apart, groups are looked through by integer compares, and a
// lane knows its best until that is elected.  (12700 cycles a token of 256 experts in 8 groups; with doubles in shared memory, a
// division by the group's size and every lane's list walked in every round 17200.)
template <typename T>
__device__ __noinline__ int elect_slowly(const RouterArgs& a, const T* logits, int lane, unsigned long long* row) {
  if (a.bias == nullptr && a.groups == 1) {   // scores rise with logits
    for (int e = lane; e < a.experts; e += 32) row[e] = (unsigned long long)order_key(Elem<T>::load1(logits + e)) << 32;
  } else {
    double m = 0.0, part_of = 1.0;   // the softmax's maximum, and one over its sum
    if (!a.sigmoid) {
      float top = -CUDART_INF_F;
      for (int e = lane; e < a.experts; e += 32) {
        const float l = Elem<T>::load1(logits + e);
        top = l > top || l != l ? l : top;
      }
      m = lanes_max(top, 32);
      double sum = 0.0;
#pragma unroll 4
      for (int e = lane; e < a.experts; e += 32) {
        const float l = Elem<T>::load1(logits + e);
        sum += l == -CUDART_INF_F ? 0.0 : exp((double)l - m);
      }
      sum = lanes_add(sum, 32);
      part_of = sum == 0.0 ? 0.0 : 1.0 / sum;
    }
#pragma unroll 4
    for (int e = lane; e < a.experts; e += 32) {
      const float l = Elem<T>::load1(logits + e);
      const double x = exp(a.sigmoid ? -(double)l : (double)l - m);
      const double v = (a.sigmoid ? __drcp_rn(1.0 + x) : x * part_of) + (a.bias != nullptr ? (double)a.bias[e] : 0.0);
      row[e] = order_key(l == -CUDART_INF_F ? -CUDART_INF : v);
    }
  }
  if (a.groups > 1) {
    __syncwarp();
    int part = 32;   // lanes that look through one group
    while (part * a.groups > 32) part >>= 1;
    const int size = a.experts / a.groups, mine = lane / part;
    unsigned long long best = 0ull, next = 0ull;
    if (mine < a.groups) {
      for (int i = lane % part; i < size; i += part) {
        const unsigned long long k = row[mine * size + i];
        next = max(next, min(best, k));
        best = max(best, k);
      }
    }
    for (int o = part >> 1; o > 0; o >>= 1) {
      const unsigned long long f = __shfl_xor_sync(0xffffffffu, best, o), n = __shfl_xor_sync(0xffffffffu, next, o);
      next = max(min(best, f), max(next, n));
      best = max(best, f);
    }
    // (the key of -inf: no second expert that is not masked; there is none at all in a group of one)
    const double sum = next <= order_key(-CUDART_INF) ? value_of(best) : value_of(best) + value_of(next);
    const unsigned long long key = order_key(__shfl_sync(0xffffffffu, sum, lane * part & 31));   // lane g ranks group g
    int ahead = 0;
    for (int g = 0; g < a.groups; ++g) {
      const unsigned long long other = __shfl_sync(0xffffffffu, key, g);
      ahead += other > key || (other == key && g < lane);
    }
    const uint32_t open = __ballot_sync(0xffffffffu, lane < a.groups && ahead < a.top_groups);
    __syncwarp();
    if (mine < a.groups && (a.bias == nullptr || !(open >> mine & 1u)))   // (without a bias the order is that of the logits again)
      for (int e = mine * size + lane % part; e < (mine + 1) * size; e += part)
        row[e] = open >> mine & 1u ? (unsigned long long)order_key(Elem<T>::load1(logits + e)) << 32 : 0ull;
  }
  __syncwarp();
  unsigned long long best = 0ull;
  int at = a.experts, elected = 0;
  bool stale = true;
  for (int j = 0; j < a.top_k; ++j) {
    if (stale) {   // (the lane's best was elected: look for the next one among its own, which no other lane writes)
      best = 0ull;
#pragma unroll 4
      for (int e = lane; e < a.experts; e += 32) {
        const unsigned long long k = row[e];
        at = k > best ? e : at;
        best = max(best, k);
      }
    }
    // the largest upper half, of those the largest lower half, of those the lowest expert
    const uint32_t upper = (uint32_t)(best >> 32), lower = (uint32_t)best;
    const bool ahead = upper == __reduce_max_sync(0xffffffffu, upper);
    const uint32_t top = __reduce_max_sync(0xffffffffu, ahead ? lower : 0u);
    const int winner = (int)__reduce_min_sync(0xffffffffu, ahead && lower == top ? (uint32_t)at : 0xffffffffu);
    stale = at == winner;
    if (stale) row[winner] = 0ull;
    if (lane == j) elected = winner;
  }
  __syncwarp();
  return elected;
}

// How far the difference of two values of the quick election may be from the true one, over 1 + |v|.  u = 2^-24.
//   sigmoid   __expf is right to (2 + 1.17 |l|) 2 u, of which s (1 - s) arrives: 1.2 u at most; 1 + e, 2 ulp of the quotient and the
//             sum with the bias: 1, 2 and |v| u.  Twice that: below 9 u + 2 u |v|.
//   softmax   expf, its argument and the quotient: below 5 u of s; the sum of 32 terms a lane and three exchanges: 37 u of s; the two
//             scores are at most 1 together: 42 u + 2 u |v|.
__device__ __forceinline__ float value_error(bool sigmoid) { return sigmoid ? 10.f / 16777216.f : 48.f / 16777216.f; }

__device__ __forceinline__ uint32_t make_key(float v, int expert) { return (order_key(v) & 0xffffff00u) | (255u - expert); }
// the largest of the values that share a key's upper 24 bits; -inf for a masked expert's
__device__ __forceinline__ float key_ceiling(uint32_t key) {
  if (key <= 0x007fffffu) return -CUDART_INF_F;
  const uint32_t u = key | 0xffu;
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

// Keeps the best LL of two falling lists in `a`, in falling order; `lost` is the largest key left out so far.
template <int LL, bool kTrack>
__device__ __forceinline__ void merge_keys(uint32_t (&a)[LL], const uint32_t (&b)[LL], uint32_t& lost) {
#pragma unroll
  for (int i = 0; i < LL; ++i) {
    if (kTrack) lost = max(lost, min(a[i], b[LL - 1 - i]));
    a[i] = max(a[i], b[LL - 1 - i]);
  }
#pragma unroll
  for (int step = LL / 2; step > 0; step >>= 1) {   // (what is left rises and falls once)
#pragma unroll
    for (int i = 0; i < LL; ++i)
      if ((i & step) == 0) sort_pair(a[i], a[i + step]);
  }
}

// Sigmoid scores as numbers: s = e^min(x,0) / (1 + e^-|x|) over e^shift.  Shares s_j / sum_S s do not depend on the shift, and with the
// largest chosen logit m in it, where that is negative, they are right however low the logits lie (e^-89 is no fp32 number).
// (The maximum over the lanes that serve a token: one instruction where that is the whole warp.)
__device__ __forceinline__ float share_shift(float x, int width) {
  float m;
  if (width == 32) {
    const uint32_t key = __reduce_max_sync(0xffffffffu, order_key(x));
    m = key >= order_key(0.f) ? 0.f : __uint_as_float(~key);
  } else {
    m = lanes_max(x, width);
  }
  return m < 0.f && m != -CUDART_INF_F ? m : 0.f;
}
__device__ __forceinline__ float sigmoid_over(float x, float shift) { return expf(fminf(x, 0.f) - shift) / (1.f + expf(-fabsf(x))); }

// The weights of the elected: lane j (of `width` that serve the token) has the j-th expert and its logit x, `chosen` for
// j < top_k.  m and z: the maximum and the sum of the softmax over all experts (not needed where it is renormalised).
template <typename T>
__device__ __forceinline__ void write_choice(const RouterArgs& a, long long at, bool chosen, int width, int expert, float x, float m, float z) {
  float s;
  if (a.sigmoid) {
    const float shift = a.renormalize ? share_shift(chosen ? x : -CUDART_INF_F, width) : 0.f;
    s = chosen ? sigmoid_over(x, shift) : 0.f;
  } else {
    if (a.renormalize) m = lanes_max(chosen ? x : -CUDART_INF_F, width);
    s = chosen && x != -CUDART_INF_F ? expf(x - m) : 0.f;
    if (!a.renormalize) s = z == 0.f ? 0.f : s / z;
  }
  if (a.renormalize) {
    const float sum = lanes_add(s, width);
    s = sum == 0.f ? 0.f : s / sum;
  }
  if (chosen) {
    Elem<T>::store1(static_cast<T*>(a.weights) + at, s * a.scale);
    a.indices[at] = expert;
  }
}

// The quick election.  A lane holds RUNS runs of RL experts and a list of LL keys (top_k <= LL).  kValues: a bias or groups take part
// (without a bias the values are there for the groups' sums, and the keys are those of the logits).
template <typename T, int RL, int RUNS, int LL, bool kValues>
__global__ void __launch_bounds__(kRouterThreads, 4) router_topk_kernel(const __grid_constant__ RouterArgs a) {
  constexpr bool kExact = !kValues && sizeof(T) == 2;
  __shared__ unsigned long long rows[kExact ? 1 : kRouterThreads / 32][kExact ? 1 : kQuickLanes * RL * RUNS];
  const int lane = threadIdx.x & 31, place = lane % kQuickLanes, warp = threadIdx.x >> 5;
  const long long warp_token = (long long)blockIdx.x * kQuickTokens + warp * (32 / kQuickLanes);
  if (warp_token >= a.tokens) return;   // (whole warps leave: the lanes of a token that is not there go along)
  const long long t = warp_token + lane / kQuickLanes;
  const bool there = t < a.tokens;
  const T* row = static_cast<const T*>(a.logits) + (there ? t : warp_token) * a.stride;
  const int part = kQuickLanes / a.groups, size = a.experts / a.groups, per = (size + part - 1) / part;   // lanes a group, experts a group, a lane
  const int group = place / part, begin = place % part * per;
  const int first = group * size + begin, mine = max(0, min(per, size - begin));
  float l[RUNS][RL];
#pragma unroll
  for (int r = 0; r < RUNS; ++r) load_run<T, RL>(row + first + r * RL, mine - r * RL, a.vector != 0, l[r]);
  float m = 0.f, z = 1.f;
  if (!a.sigmoid && (kValues || !a.renormalize)) {   // the softmax's maximum and sum
    m = l[0][0];
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int i = 0; i < RL; ++i) m = l[r][i] > m || l[r][i] != l[r][i] ? l[r][i] : m;
    m = lanes_max(m, kQuickLanes);
    z = 0.f;
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int i = 0; i < RL; ++i) z += l[r][i] == -CUDART_INF_F ? 0.f : expf(l[r][i] - m);
    z = lanes_add(z, kQuickLanes);
  }
  auto value = [&](float x, float b) -> float {
    if (!kValues || x == -CUDART_INF_F) return x;
    return (a.sigmoid ? quick_sigmoid(x) : __fdividef(expf(x - m), z)) + b;
  };
  const bool grouped = kValues && a.groups > 1, by_logit = !kValues || a.bias == nullptr;
  const bool exact = by_logit && sizeof(T) == 2;          // the keys tell any two experts apart
  float best_v = -CUDART_INF_F, next_v = -CUDART_INF_F;   // the two largest values of this lane's part of a group
  uint32_t list[LL], lost = 0u;
#pragma unroll
  for (int i = 0; i < LL; ++i) list[i] = 0u;
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    uint32_t key[RL], best[LL];
    float bias[RL];
#pragma unroll
    for (int i = 0; i < RL; ++i) bias[i] = 0.f;
    if (kValues && a.bias != nullptr) load_run<float, RL>(a.bias + first + r * RL, mine - r * RL, a.vector_bias != 0, bias);
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      const int e = first + r * RL + i;
      const bool has = r * RL + i < mine;
      const float v = has ? value(l[r][i], bias[i]) : -CUDART_INF_F;
      key[i] = has ? make_key(by_logit ? l[r][i] : v, e) : 0u;
      if (grouped) {
        next_v = fmaxf(next_v, fminf(best_v, v));
        best_v = fmaxf(best_v, v);
      }
    }
    sort_keys<RL>(key);
#pragma unroll
    for (int i = 0; i < LL; ++i) best[i] = i < RL ? key[i] : 0u;
    if (RL > LL && !kExact) lost = max(lost, key[LL < RL ? LL : 0]);
    if (r == 0) {
#pragma unroll
      for (int i = 0; i < LL; ++i) list[i] = best[i];
    } else {
      merge_keys<LL, !kExact>(list, best, lost);
    }
  }
  bool sure = true;
  if (grouped) {
    for (int o = part >> 1; o > 0; o >>= 1) {
      const float f = __shfl_xor_sync(0xffffffffu, best_v, o), n = __shfl_xor_sync(0xffffffffu, next_v, o);
      next_v = fmaxf(fminf(best_v, f), fmaxf(next_v, n));
      best_v = fmaxf(best_v, f);
    }
    const float sum = next_v == -CUDART_INF_F ? best_v : best_v + next_v;
    const float slack = best_v == -CUDART_INF_F ? 0.f : value_error(a.sigmoid) * (2.f + fabsf(best_v) + (next_v == -CUDART_INF_F ? 0.f : fabsf(next_v)));
    int ahead = 0;
    for (int g = 0; g < a.groups; ++g) {
      const float other = __shfl_sync(0xffffffffu, sum, g * part, kQuickLanes);
      ahead += other > sum || (other == sum && g < group);
    }
    const bool open = ahead < a.top_groups;
    if (a.top_groups < a.groups) {   // the narrowest of the gaps between an open group and a closed one
      const float in = -lanes_max(open ? -sum : -CUDART_INF_F, kQuickLanes), out = lanes_max(open ? -CUDART_INF_F : sum, kQuickLanes);
      const float most = lanes_max(slack, kQuickLanes);
      // (no NaN, in a logit or a bias or from a softmax over +inf: the maxima pass it by)
      sure = (in - out > most || (in == -CUDART_INF_F && out == -CUDART_INF_F)) && list[0] < 0xffffff00u && z == z;
    }
    if (!open) {
#pragma unroll
      for (int i = 0; i < LL; ++i) list[i] = 0u;
      lost = 0u;
    }
  }
#pragma unroll
  for (int o = 1; o < kQuickLanes; o <<= 1) {
    uint32_t other[LL];
#pragma unroll
    for (int i = 0; i < LL; ++i) other[i] = __shfl_xor_sync(0xffffffffu, list[i], o);
    if (!kExact) lost = max(lost, __shfl_xor_sync(0xffffffffu, lost, o));
    merge_keys<LL, !kExact>(list, other, lost);
  }
  uint32_t won = 0u;   // this lane's of the elected
#pragma unroll
  for (int i = 0; i < LL; ++i)
    if (place == i) won = list[i];
  const bool chosen = there && place < a.top_k;
  int expert = 255 - (int)(won & 255u);
  float x = chosen && won != 0u ? Elem<T>::load1(row + expert) : -CUDART_INF_F;
  if (!kExact) {
    float b = 0.f, v = x;
    if (!by_logit && chosen) {
      b = a.bias[expert];
      v = value(x, b);
    }
    const float pv = __shfl_up_sync(0xffffffffu, v, 1, kQuickLanes), px = __shfl_up_sync(0xffffffffu, x, 1, kQuickLanes);
    const float pb = __shfl_up_sync(0xffffffffu, b, 1, kQuickLanes);
    const float error = by_logit ? 0.f : value_error(a.sigmoid) * (1.f + fabsf(v));
    if (!exact && place > 0 && chosen) sure = sure && ((x == -CUDART_INF_F && px == -CUDART_INF_F) || (px == x && pb == b) || pv - v > error);
    if (!exact && place == a.top_k - 1) {   // the best of those left out: no one's value is above its key's
      uint32_t behind = lost;
#pragma unroll
      for (int i = 1; i < LL; ++i)
        if (a.top_k == i) behind = list[i];
      const float next = key_ceiling(behind);
      sure = sure && (behind == 0u || (v == -CUDART_INF_F && next == -CUDART_INF_F) || v - next > error);
    }
    const uint32_t doubtful = __ballot_sync(0xffffffffu, there && !sure);
    for (int q = 0; q < 32 / kQuickLanes; ++q) {
      if ((doubtful >> (q * kQuickLanes) & 0xffu) == 0u) continue;
      const T* other = static_cast<const T*>(a.logits) + (warp_token + q) * a.stride;
      const int found = __shfl_sync(0xffffffffu, elect_slowly<T>(a, other, lane, rows[warp]), place);
      if (lane / kQuickLanes == q) expert = found;
      if (lane / kQuickLanes == q && chosen) x = Elem<T>::load1(row + expert);
    }
  }
  write_choice<T>(a, t * a.top_k + place, chosen, kQuickLanes, expert, x, m, z);
}

// Any groups and top_k: one warp a token, the slow election.
template <typename T>
__global__ void __launch_bounds__(kRouterThreads) router_topk_any_kernel(const __grid_constant__ RouterArgs a) {
  __shared__ unsigned long long rows[kRouterThreads / 32][kRouterMaxExperts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = (long long)blockIdx.x * (kRouterThreads / 32) + warp;
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  float m = 0.f, z = 1.f;
  if (!a.sigmoid && !a.renormalize) {
    m = -CUDART_INF_F;
    for (int e = lane; e < a.experts; e += 32) {
      const float l = Elem<T>::load1(row + e);
      m = l > m || l != l ? l : m;
    }
    m = lanes_max(m, 32);
    z = 0.f;
    for (int e = lane; e < a.experts; e += 32) {
      const float l = Elem<T>::load1(row + e);
      z += l == -CUDART_INF_F ? 0.f : expf(l - m);
    }
    z = lanes_add(z, 32);
  }
  const int expert = elect_slowly<T>(a, row, lane, rows[warp]);
  const bool chosen = lane < a.top_k;
  write_choice<T>(a, t * a.top_k + lane, chosen, 32, expert, chosen ? Elem<T>::load1(row + expert) : -CUDART_INF_F, m, z);
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

// With d_j = scale * dw_j and r_j = s_j / sum_S s:
//   sigmoid   dl_j = d_j s_j (1 - s_j) for the chosen, 0 elsewhere; renormalised that is r_j (d_j - sum_S d r) (1 - s_j)
//   softmax   dl_i = s_i (d_i - sum_S d s), d_i = 0 where i is not chosen; renormalised that is r_j (d_j - sum_S d r), 0 elsewhere
//
// W lanes serve a token (8, or 32 where top_k is above 8): lane j has the j-th chosen expert, and all of them write the row, RUNS
// runs of RL experts a lane.
template <typename T, int RL, int RUNS, int W>
__global__ void __launch_bounds__(kRouterThreads) router_topk_bwd_kernel(const __grid_constant__ RouterBwdArgs a) {
  const int lane = threadIdx.x & 31, place = lane % W;
  const long long warp_token = ((long long)blockIdx.x * (kRouterThreads / 32) + (threadIdx.x >> 5)) * (32 / W);
  if (warp_token >= a.tokens) return;   // (whole warps leave)
  const long long t = warp_token + lane / W;
  const bool there = t < a.tokens;
  const T* row = static_cast<const T*>(a.logits) + (there ? t : warp_token) * a.stride;
  int e = -1;
  float lj = -CUDART_INF_F, d = 0.f;
  if (there && place < a.top_k) {
    const long long index = a.indices[t * a.top_k + place];
    e = index >= 0 && index < a.experts ? (int)index : -1;
    if (e >= 0) lj = Elem<T>::load1(row + e);
    d = Elem<T>::load1(static_cast<const T*>(a.dweights) + t * a.top_k + place) * a.scale;
  }
  float g[RUNS][RL], chosen;   // the gradients of this lane's runs; of its chosen expert
#pragma unroll
  for (int r = 0; r < RUNS; ++r)
#pragma unroll
    for (int i = 0; i < RL; ++i) g[r][i] = 0.f;
  if (a.sigmoid) {
    const float x = expf(-fabsf(lj)), rest = (lj >= 0.f ? x : 1.f) / (1.f + x);   // 1 - s (no overflow on either side)
    if (a.renormalize) {
      const float s = sigmoid_over(lj, share_shift(lj, W));   // (0 where there is no expert)
      const float sum = lanes_add(s, W);
      const float r = sum == 0.f ? 0.f : s / sum;
      chosen = r * (d - lanes_add(e >= 0 ? d * r : 0.f, W)) * rest;
    } else {
      chosen = d * sigmoid_over(lj, 0.f) * rest;
    }
  } else if (a.renormalize) {
    const float m = lanes_max(lj, W);
    const float s = lj == -CUDART_INF_F ? 0.f : expf(lj - m);
    const float sum = lanes_add(s, W);
    const float r = sum == 0.f ? 0.f : s / sum;
    chosen = r * (d - lanes_add(e >= 0 ? d * r : 0.f, W));
  } else {
    float m = -CUDART_INF_F, z = 0.f;
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      const int first = (r * W + place) * RL, n = a.experts - first;
      load_run<T, RL>(row + first, n, a.vector_in != 0 && n >= RL, g[r]);
#pragma unroll
      for (int i = 0; i < RL; ++i) m = g[r][i] > m || g[r][i] != g[r][i] ? g[r][i] : m;
    }
    m = lanes_max(m, W);
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int i = 0; i < RL; ++i) {
        g[r][i] = g[r][i] == -CUDART_INF_F ? 0.f : expf(g[r][i] - m);
        z += g[r][i];
      }
    z = lanes_add(z, W);
    const float s = lj == -CUDART_INF_F || z == 0.f ? 0.f : expf(lj - m) / z;
    const float dot = lanes_add(e >= 0 ? d * s : 0.f, W);
    chosen = s * (d - dot);
    const float back = z == 0.f ? 0.f : -dot / z;
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int i = 0; i < RL; ++i) g[r][i] *= back;
  }
  // the whole row first, then the chosen experts over it (stores of one warp in this order)
  T* out = static_cast<T*>(a.dlogits) + t * a.experts;
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    const int first = (r * W + place) * RL, n = there ? a.experts - first : 0;
    store_run<T, RL>(out + first, n, a.vector_out != 0 && n >= RL, g[r]);
  }
  __syncwarp();
  if (e >= 0) Elem<T>::store1(out + e, chosen);
}

}  // namespace b200moe
