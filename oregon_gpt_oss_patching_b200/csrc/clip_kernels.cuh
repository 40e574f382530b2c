// The global norm of many gradients, clipping by it, and the state-free SGD update with the clip folded in.
//
//   n = sqrt(sum over all tensors of g^2),  c = min(1, max_norm / (n + 1e-6)),  g <- round(c g)   or   p <- round(p - lr c g)
//
// Two launches: `grad_sumsq_kernel` reads every gradient once and leaves one partial sum a CTA; each CTA of the second
// kernel adds the same partials in the same order, so all of them hold the same c without a third launch, a counter or
// atomics, and writes back (nothing, where c = 1).  The second may start while the first runs out, and goes through its
// tensors backwards, since what the first read last is still in L2.  (Lists of more than kClipTensors take a launch of each kernel for every
// so many, in the list's order; of those only the last launch's tensors can still be there.)
//
// Both are bound by HBM: clipping cannot do without reading the gradients twice (unless they fit in L2) and writing them once;
// the folded update reads gradients twice and parameters once and writes the parameters, where clipping first and updating
// then moves half as much again.  One decoder layer's 823 M bf16 gradients: norm 232 us (7.1 TB/s), clip 780 us (6.3 TB/s, the
// second read included), update 985 us (6.7 TB/s).  (Loads one word at a time between the stores, which the compiler must keep
// in order: update 1212 us.)
//
// The tensors' addresses and sizes travel as a kernel parameter (no copy to the device, nothing to keep alive, nothing for a
// captured graph to find changed).  Work is cut into chunks of kChunkWords 16-byte words of the 16-byte grid that covers a
// tensor; a word at a tensor's end that it shares with other memory is moved element by element.
#pragma once
#include "elem_types.cuh"

namespace b200train {

constexpr int kClipThreads = 256;
constexpr int kClipTensors = 256;     // of one launch
constexpr int kChunkWords = 2048;     // 32 KB

struct ClipTable {
  void* grad[kClipTensors];
  void* param[kClipTensors];
  long long count[kClipTensors];      // elements
  unsigned first[kClipTensors];       // a tensor's first chunk
  unsigned char dtype[kClipTensors];
  int tensors;
  unsigned chunks;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum over the CTA, in every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipThreads / 32];
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum((threadIdx.x & 31) < kClipThreads / 32 ? part[threadIdx.x & 31] : 0.0);
}

// The tensor that holds a chunk: the last one whose first chunk is not behind it.
__device__ __forceinline__ int tensor_of(const ClipTable& t, unsigned chunk) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A chunk of one tensor: words [begin, end) of the 16-byte grid, the tensor's elements being [off, off + count) of that grid.
template <typename T>
struct Chunk {
  static constexpr int N = Elem<T>::N;
  long long begin, end, off, last;   // last = off + count
  __device__ __forceinline__ Chunk(const void* grad, long long count, unsigned index) {
    off = (long long)((reinterpret_cast<uintptr_t>(grad) & 15u) / sizeof(T));
    last = off + count;
    const long long words = (last + N - 1) / N;
    begin = (long long)index * kChunkWords;
    end = begin + kChunkWords < words ? begin + kChunkWords : words;
  }
  __device__ __forceinline__ bool whole() const { return end - begin == kChunkWords && inside(begin) && inside(end - 1); }
  __device__ __forceinline__ bool inside(long long w) const { return w * N >= off && (w + 1) * N <= last; }
  // element e of word w relative to the tensor's first element, and whether the tensor has it
  __device__ __forceinline__ long long at(long long w, int e) const { return w * N + e - off; }
  __device__ __forceinline__ bool has(long long w, int e) const { return w * N + e >= off && w * N + e < last; }
  __device__ __forceinline__ void load(const T* p, long long w, bool vector, float* f) const {
    if (vector && inside(w)) {
      unpack<T>(*reinterpret_cast<const uint4*>(p + at(w, 0)), f);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = has(w, e) ? Elem<T>::load1(p + at(w, e)) : 0.f;
    }
  }
  __device__ __forceinline__ void store(T* p, long long w, bool vector, const float* f) const {
    if (vector && inside(w)) {
      *reinterpret_cast<uint4*>(p + at(w, 0)) = pack<T>(f);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (has(w, e)) Elem<T>::store1(p + at(w, e), f[e]);
    }
  }
};

// A chunk that has all its words, none of them shared: its words are loaded kBatch at a time before any is used or stored.
constexpr int kBatch = 4;
static_assert(kChunkWords % (kClipThreads * kBatch) == 0, "a whole chunk is whole batches");

// The sum of the squares of a 16-byte word's elements.  It is made in fp32, a tree of two (fp32 elements) or three additions, and all
// above it in fp64: the sum is right to 3 * 2^-24 whatever the sizes and the order of its terms.  (fp64 from the squares on, which is
// 2^-24 for fp32 elements and exact for others, is bound by the conversions: 823 M bf16 237 to 241 us instead of 232, 20 M in L2 12.9
// instead of 9.2.  fp32 for all of a thread's words in a chunk, up to 64 squares, costs the same as this and may be off by 64 * 2^-24.)
template <int N>
__device__ __forceinline__ double word_sumsq(const F2 (&f)[N / 2]) {
  F2 p[N / 2];
#pragma unroll
  for (int e = 0; e < N / 2; ++e) p[e] = mul2(f[e], f[e]);
#pragma unroll
  for (int n = N / 4; n > 0; n /= 2) {
#pragma unroll
    for (int e = 0; e < n; ++e) p[e] = add2(p[e], p[e + n]);
  }
  const float2 s = split2(p[0]);
  return (double)(s.x + s.y);
}

template <typename T>
__device__ __forceinline__ double chunk_sumsq(const void* grad, long long count, unsigned index) {
  constexpr int N = Elem<T>::N;
  const Chunk<T> c(grad, count, index);
  const T* g = static_cast<const T*>(grad);
  double sum = 0.0;
  if (c.whole()) {
    const uint4* w = reinterpret_cast<const uint4*>(g + c.at(c.begin, 0)) + threadIdx.x;
    uint4 v[kChunkWords / kClipThreads];
#pragma unroll
    for (int i = 0; i < kChunkWords / kClipThreads; ++i) v[i] = w[i * kClipThreads];
#pragma unroll
    for (int i = 0; i < kChunkWords / kClipThreads; ++i) {
      F2 f[N / 2];
      unpack<T>(v[i], f);
      sum += word_sumsq<N>(f);
    }
  } else {
    for (long long w = c.begin + threadIdx.x; w < c.end; w += kClipThreads) {
      float f[N];
      c.load(g, w, true, f);
      F2 pairs[N / 2];
#pragma unroll
      for (int e = 0; e < N; e += 2) pairs[e / 2] = make2(f[e], f[e + 1]);
      sum += word_sumsq<N>(pairs);
    }
  }
  return sum;
}

__global__ void __launch_bounds__(kClipThreads) grad_sumsq_kernel(const __grid_constant__ ClipTable t, double* partials) {
  asm volatile("griddepcontrol.launch_dependents;");
  double sum = 0.0;
  for (unsigned chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int i = tensor_of(t, chunk);
    const unsigned index = chunk - t.first[i];
    double s;
    if (t.dtype[i] == 0) s = chunk_sumsq<__nv_bfloat16>(t.grad[i], t.count[i], index);
    else if (t.dtype[i] == 1) s = chunk_sumsq<__half>(t.grad[i], t.count[i], index);
    else s = chunk_sumsq<float>(t.grad[i], t.count[i], index);
    sum += s;
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

template <typename T, bool kUpdate>
__device__ __forceinline__ void chunk_apply(void* grad, void* param, long long count, unsigned index, float scale) {
  constexpr int N = Elem<T>::N;
  const Chunk<T> c(grad, count, index);
  T* g = static_cast<T*>(grad);
  T* p = static_cast<T*>(param);
  // a parameter that lies otherwise on the 16-byte grid than its gradient is moved element by element
  const bool same = !kUpdate || ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(param)) & 15u) == 0;
  const F2 times = make2(kUpdate ? -scale : scale, kUpdate ? -scale : scale);
  if (same && c.whole()) {
    const uint4* w = reinterpret_cast<const uint4*>(g + c.at(c.begin, 0)) + threadIdx.x;
    uint4* out = kUpdate ? reinterpret_cast<uint4*>(p + c.at(c.begin, 0)) + threadIdx.x : const_cast<uint4*>(w);
#pragma unroll 1
    for (int k = 0; k < kChunkWords / kClipThreads; k += kBatch) {
      uint4 v[kBatch], q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        v[i] = w[(k + i) * kClipThreads];
        if (kUpdate) q[i] = out[(k + i) * kClipThreads];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        F2 f[N / 2], r[N / 2];
        unpack<T>(v[i], f);
        if (kUpdate) unpack<T>(q[i], r);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) r[e] = kUpdate ? fma2(times, f[e], r[e]) : mul2(times, f[e]);
        out[(k + i) * kClipThreads] = pack<T>(r);
      }
    }
    return;
  }
  for (long long w = c.begin + threadIdx.x; w < c.end; w += kClipThreads) {
    float f[N], q[N];
    c.load(g, w, true, f);
    if (kUpdate) {
      c.load(p, w, same, q);
#pragma unroll
      for (int e = 0; e < N; ++e) q[e] = fmaf(-scale, f[e], q[e]);
      c.store(p, w, same, q);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] *= scale;
      c.store(g, w, true, f);
    }
  }
}

// kUpdate: p <- p - lr c g, otherwise g <- c g.  `norm` gets sqrt of the sum of the partials.
template <bool kUpdate>
__global__ void __launch_bounds__(kClipThreads)
clip_apply_kernel(const __grid_constant__ ClipTable t, const double* partials, int parts, float max_norm, float lr, float* norm) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kClipThreads) sum += partials[i];
  const float n = (float)sqrt(block_sum(sum));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm != nullptr) *norm = n;
  float scale = isinf(max_norm) ? 1.f : max_norm / (n + 1e-6f);   // (no limit: nothing is scaled, whatever the norm)
  if (scale >= 1.f) {   // (not where it is NaN: that goes into the gradients)
    if (!kUpdate) return;
    scale = 1.f;
  }
  if (kUpdate) scale *= lr;
  // from the last chunk to the first: the last ones read by the kernel before are still in L2
  for (unsigned k = blockIdx.x; k < t.chunks; k += gridDim.x) {
    const unsigned chunk = t.chunks - 1 - k;
    const int i = tensor_of(t, chunk);
    const unsigned index = chunk - t.first[i];
    if (t.dtype[i] == 0) chunk_apply<__nv_bfloat16, kUpdate>(t.grad[i], t.param[i], t.count[i], index, scale);
    else if (t.dtype[i] == 1) chunk_apply<__half, kUpdate>(t.grad[i], t.param[i], t.count[i], index, scale);
    else chunk_apply<float, kUpdate>(t.grad[i], t.param[i], t.count[i], index, scale);
  }
}

// norm <- sqrt of the sum of the partials (the norm alone is asked for).
__global__ void __launch_bounds__(kClipThreads) grad_norm_kernel(const double* partials, int parts, float* norm) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kClipThreads) sum += partials[i];
  sum = block_sum(sum);
  if (threadIdx.x == 0) *norm = (float)sqrt(sum);
}

}  // namespace b200train
