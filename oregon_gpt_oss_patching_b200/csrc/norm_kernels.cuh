// The residual sum with its RMS norm and their gradient, each as one pass over the rows.
//
// Forward:   h = round(x + r),  y = w * h * rstd,  rstd = 1 / sqrt(mean(h^2) + eps)
// Backward:  with n = h * rstd, g = dy * w:   dx = dh + rstd * (g - n * mean(g * n)),   dw = sum over the rows of dy * n
//
// GptOssRMSNorm.forward (transformers/models/gpt_oss/modeling_gpt_oss.py:57-63) runs eight elementwise passes and a
// reduction over an fp32 copy of the row; here a row is read once into registers, reduced, and written once, so both
// kernels are bound by HBM: four tensors cross it in either direction of the pass with a residual.
//
// A row belongs to a "row lane": blockDim.x threads (whole warps) that meet at a named barrier of their own, so that
// the blockDim.y row lanes of a CTA drift apart and one's loads cover another's reduction.  A thread holds VPT 16-byte
// words of each tensor.  Rows whose length is no multiple of 16 bytes (kShift) are walked in the 16-byte words that
// cover them: the words at a row's two ends are shared with its neighbours and moved element by element, the others whole.
// The row's place inside its first word depends on the row's index modulo 8 alone, so a lane that steps by a multiple
// of 8 rows owns the same columns in every row: weights and dw sums stay in registers there too.
#pragma once
#include "elem_types.cuh"

namespace b200train {

constexpr int kNormMaxLanes = 8;       // row lanes of a CTA: named barriers 1 .. 8
constexpr int kNormMaxThreads = 512;   // of a CTA, in all its row lanes
constexpr int kNormMaxWarps = kNormMaxThreads / 32;

__device__ __forceinline__ void lane_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Where a row lies: `off` elements into its first 16-byte word, `words` words in all.
template <typename T, bool kShift>
struct RowSpan {
  static constexpr int N = Elem<T>::N;
  int off, cols, words;
  __device__ __forceinline__ RowSpan(long long row, int cols_) : cols(cols_) {
    off = kShift ? (int)((row * cols_) & (N - 1)) : 0;
    words = (off + cols_ + N - 1) / N;
  }
  __device__ __forceinline__ bool inside(int c) const { return !kShift || (c * N >= off && (c + 1) * N <= off + cols); }
  // `row` points at the row's first element
  __device__ __forceinline__ void load(const T* row, int c, float* f) const {
    const T* p = row - off + c * N;
    if (inside(c)) {
      unpack<T>(*reinterpret_cast<const uint4*>(p), f);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int col = c * N + e - off;
        f[e] = (col >= 0 && col < cols) ? Elem<T>::load1(p + e) : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int c, const float* f) const {
    T* p = row - off + c * N;
    if (inside(c)) {
      *reinterpret_cast<uint4*>(p) = pack<T>(f);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int col = c * N + e - off;
        if (col >= 0 && col < cols) Elem<T>::store1(p + e, f[e]);
      }
    }
  }
  template <typename W>
  __device__ __forceinline__ void load_weight(const W* w, int c, float* f) const {
    if constexpr (!kShift) {
#pragma unroll
      for (int e = 0; e < N; e += Elem<W>::N) unpack<W>(__ldg(reinterpret_cast<const uint4*>(w + c * N + e)), f + e);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int col = c * N + e - off;
        f[e] = (col >= 0 && col < cols) ? Elem<W>::load1(w + col) : 0.f;
      }
    }
  }
};

template <typename T, typename W>
struct NormArgs {
  const T *x, *r;
  const W* w;
  T *y, *h;
  long long x_stride, r_stride, rows;
  int cols;
  float eps;
};

template <typename T, typename W, int VPT, bool kShift>
__global__ void __launch_bounds__(kNormMaxThreads) add_rms_norm_kernel(const NormArgs<T, W> a) {
  constexpr int N = Elem<T>::N;
  __shared__ float part[kNormMaxLanes][kNormMaxWarps];
  const int tid = threadIdx.x, lane = threadIdx.y, warps = blockDim.x >> 5;
  const long long row = (long long)blockIdx.x * blockDim.y + lane;
  if (row >= a.rows) return;   // the whole row lane leaves: its barrier is its own
  const RowSpan<T, kShift> span(row, a.cols);
  const T* x = a.x + row * a.x_stride;
  float v[VPT][N];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = tid + i * blockDim.x;
    if (c < span.words) span.load(x, c, v[i]);
  }
  if (a.r != nullptr) {
    const T* r = a.r + row * a.r_stride;
    T* h = a.h + row * a.cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * blockDim.x;
      if (c < span.words) {
        float q[N];
        span.load(r, c, q);
#pragma unroll
        for (int e = 0; e < N; ++e) v[i][e] = Elem<T>::round(v[i][e] + q[e]);
        span.store(h, c, v[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (tid + i * (int)blockDim.x < span.words) {
#pragma unroll
      for (int e = 0; e < N; ++e) ss = fmaf(v[i][e], v[i][e], ss);
    }
  ss = warp_sum(ss);
  if (warps > 1) {
    if ((tid & 31) == 0) part[lane][tid >> 5] = ss;
    lane_barrier(1 + lane, blockDim.x);
    ss = warp_sum((tid & 31) < warps ? part[lane][tid & 31] : 0.f);
  }
  const float rstd = rsqrtf(ss / (float)a.cols + a.eps);
  T* y = a.y + row * a.cols;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = tid + i * blockDim.x;
    if (c < span.words) {
      float w[N];
      span.load_weight(a.w, c, w);
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = v[i][e] * rstd * w[e];
      span.store(y, c, w);
    }
  }
}

template <typename T, typename W>
struct NormBwdArgs {
  const T *dy, *dh, *h;
  const W* w;
  T* dx;
  float* partial;   // (gridDim.x, cols): this CTA's part of dw, or nullptr
  long long dy_stride, dh_stride, h_stride, rows;
  int cols;
  float eps;
};

// Persistent: row lane L of all gridDim.x * blockDim.y takes the rows L, L + lanes, ... and keeps the weights and its part
// of dw in registers.  The row lanes of a CTA add their parts in lane order through shared memory (blockDim.y * cols floats).
template <typename T, typename W, int VPT, bool kShift>
__global__ void __launch_bounds__(kNormMaxThreads) add_rms_norm_bwd_kernel(const NormBwdArgs<T, W> a) {
  constexpr int N = Elem<T>::N;
  extern __shared__ float dw_part[];
  __shared__ float2 part[2][kNormMaxLanes][kNormMaxWarps];
  const int tid = threadIdx.x, lane = threadIdx.y, warps = blockDim.x >> 5;
  const long long first = (long long)blockIdx.x * blockDim.y + lane, step = (long long)gridDim.x * blockDim.y;
  const RowSpan<T, kShift> span(first, a.cols);   // (step is a multiple of 8: the same place in every row of this lane)
  float w[VPT][N], dw[VPT][N];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = tid + i * blockDim.x;
#pragma unroll
    for (int e = 0; e < N; ++e) w[i][e] = dw[i][e] = 0.f;
    if (c < span.words) span.load_weight(a.w, c, w[i]);
  }
  int turn = 0;
  for (long long row = first; row < a.rows; row += step, turn ^= 1) {
    const T* hr = a.h + row * a.h_stride;
    const T* dyr = a.dy + row * a.dy_stride;
    float h[VPT][N], dy[VPT][N];
    float ss = 0.f, sg = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * blockDim.x;
      if (c < span.words) {
        span.load(hr, c, h[i]);
        span.load(dyr, c, dy[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + i * (int)blockDim.x < span.words) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          ss = fmaf(h[i][e], h[i][e], ss);
          sg = fmaf(dy[i][e] * w[i][e], h[i][e], sg);
        }
      }
    ss = warp_sum(ss);
    sg = warp_sum(sg);
    if (warps > 1) {
      if ((tid & 31) == 0) part[turn][lane][tid >> 5] = make_float2(ss, sg);
      lane_barrier(1 + lane, blockDim.x);   // (the other buffer is free again: every thread has read it before it came here)
      const float2 p = (tid & 31) < warps ? part[turn][lane][tid & 31] : make_float2(0.f, 0.f);
      ss = warp_sum(p.x);
      sg = warp_sum(p.y);
    }
    const float rstd = rsqrtf(ss / (float)a.cols + a.eps);
    const float mean_gn = sg * rstd / (float)a.cols;
    const T* dhr = a.dh != nullptr ? a.dh + row * a.dh_stride : nullptr;
    T* dx = a.dx + row * a.cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * blockDim.x;
      if (c < span.words) {
        float o[N];
        if (dhr != nullptr) {
          span.load(dhr, c, o);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float n = h[i][e] * rstd;
          dw[i][e] = fmaf(dy[i][e], n, dw[i][e]);
          o[e] += rstd * (dy[i][e] * w[i][e] - n * mean_gn);
        }
        span.store(dx, c, o);
      }
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = tid + i * blockDim.x;
    if (c < span.words) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int col = c * N + e - span.off;
        if (!kShift || (col >= 0 && col < a.cols)) dw_part[lane * a.cols + col] = dw[i][e];
      }
    }
  }
  __syncthreads();
  for (int col = lane * blockDim.x + tid; col < a.cols; col += blockDim.x * blockDim.y) {
    float s = dw_part[col];
    for (int l = 1; l < blockDim.y; ++l) s += dw_part[l * a.cols + col];
    a.partial[(long long)blockIdx.x * a.cols + col] = s;
  }
}

// dw[c] = sum over the CTAs' parts, in a fixed order: 32 columns a CTA, 32 parts at a time.
template <typename W>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* __restrict__ partial, W* __restrict__ dw, int parts, int cols) {
  __shared__ float s[32][33];
  const int x = threadIdx.x, y = threadIdx.y, c = blockIdx.x * 32 + x;
  float acc = 0.f;
  if (c < cols)
    for (int p = y; p < parts; p += 32) acc += partial[(long long)p * cols + c];
  s[y][x] = acc;
  __syncthreads();
  acc = warp_sum(s[x][y]);
  if (x == 0 && blockIdx.x * 32 + y < cols) Elem<W>::store1(dw + blockIdx.x * 32 + y, acc);
}

}  // namespace b200train
