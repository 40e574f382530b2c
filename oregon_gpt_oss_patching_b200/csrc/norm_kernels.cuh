// The residual sum with its RMS norm and their gradient, each as one pass over the rows.
//
// Forward:   h = round(x + r),  y = w * h * rstd,  rstd = 1 / sqrt(mean(h^2) + eps)
// Backward:  with n = h * rstd, g = dy * w:   dx = dh + rstd * (g - n * mean(g * n)),   dw = sum over the rows of dy * n
//
// GptOssRMSNorm.forward (transformers/models/gpt_oss/modeling_gpt_oss.py:57-63) runs eight elementwise passes and a
// reduction over an fp32 copy of the row; here a row is read once, reduced, and written once, so both kernels are bound by
// HBM: four tensors cross it in either direction of the pass with a residual.  8192 x 2880 bf16: forward 35 us (5.4 TB/s; a copy
// of as many bytes takes 36 us), backward 33 us (5.7 TB/s) and 5 us for the weight's gradient.
//
// Both kernels are persistent.  A row belongs to a "row lane": blockDim.x threads (8, 16, or whole warps) that meet at a
// named barrier of their own where they are more than a warp, so the blockDim.y row lanes of a CTA drift apart.  A thread
// holds VPT 16-byte words of a row, the same columns in every row, so that weights and dw sums stay in registers, and copies
// the words of the rows to come into shared memory of its own (cp.async): no barrier guards the ring, no register waits
// for HBM, and one or two rows a lane are always on their way (none where fp32 rows fill the ring: above 13312 columns with two
// tensors, 9216 with three; 1024 x 16384 fp32: forward 49 us, backward 53 us, 5.5 and 5.0 TB/s).  (One CTA of 512 threads an SM.  Rows held in registers and read
// as they are needed: 49 and 140 us.  The ring with scalar arithmetic: 37 and 33 us, and 60 % of the issue slots taken; pairs
// of fp32 values an instruction halve that.)
//
// Rows whose length is no multiple of 16 bytes (kShift) are walked in the 16-byte words that cover them; the words at a row's
// ends are shared with its neighbours: what lies outside the row is read and dropped, and the row's part is written element by
// element.  The row's place inside its first word depends on its index modulo 8 alone, and a lane steps by a multiple of 8
// rows there, so its columns stay the same.
#pragma once
#include "elem_types.cuh"

namespace b200train {

constexpr int kNormMaxThreads = 512;   // of a CTA, in all its row lanes
constexpr int kNormMaxWarps = kNormMaxThreads / 32;
constexpr int kNormBarriers = 15;      // row lanes of more than a warp: named barriers 1 .. 15

__device__ __forceinline__ void lane_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most stages - 1 of the thread's groups are on their way
__device__ __forceinline__ void copy_async_wait(int stages) {
  if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (stages >= 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// What one thread has of its row lane's rows: the words tid, tid + blockDim.x, ... of each, `live` of them inside the row;
// rows `row`, `row + step`, ...  A row starts `off` elements into its first word.
template <typename T, int VPT, bool kShift>
struct RowLane {
  static constexpr int N = Elem<T>::N;
  long long row, warp_row, step;   // warp_row: the first row of the warp, by which its threads leave the loop together
  int off, cols, tid, lane, warps, words;
  uint32_t ring, word_bytes;       // this thread's first slot of the ring, and from one word's slot to the next
  __device__ __forceinline__ RowLane(int cols_, const uint4* shared) : cols(cols_) {
    tid = threadIdx.x;
    lane = threadIdx.y;
    warps = blockDim.x >> 5;   // 0: less than a warp
    const int linear = lane * blockDim.x + tid;
    row = (long long)blockIdx.x * blockDim.y + lane;
    warp_row = row - (warps == 0 ? (linear & 31) / (int)blockDim.x : 0);
    step = (long long)gridDim.x * blockDim.y;
    off = kShift ? (int)((row * cols) & (N - 1)) : 0;
    words = (off + cols + N - 1) / N;
    word_bytes = blockDim.x * blockDim.y * 16;
    ring = (uint32_t)__cvta_generic_to_shared(shared) + linear * 16;
  }
  __device__ __forceinline__ int word(int i) const { return tid + i * blockDim.x; }
  __device__ __forceinline__ bool live(int i) const { return word(i) < words; }
  __device__ __forceinline__ int col(int i, int e) const { return word(i) * N + e - off; }
  __device__ __forceinline__ bool has(int i, int e) const { return !kShift || (unsigned)col(i, e) < (unsigned)cols; }
  __device__ __forceinline__ bool inside(int i) const { return !kShift || (has(i, 0) && has(i, N - 1)); }
  // this thread's words of the row that starts at p into the ring; `left`: elements from there to the tensor's end (nothing
  // behind it is read)
  __device__ __forceinline__ void fetch(uint32_t slot, const T* p, long long left) const {
    const T* q = p + (tid * N - off);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (live(i)) {
        if (kShift) {
          const long long rest = (left - col(i, 0)) * (long long)sizeof(T);
          copy_async16(slot + i * word_bytes, q + i * (int)blockDim.x * N, rest < 16 ? (int)rest : 16);
        } else {
          copy_async16(slot + i * word_bytes, q + i * (int)blockDim.x * N);
        }
      }
  }
  __device__ __forceinline__ void get(uint32_t slot, int i, F2* f) const {
    const uint4 v = load_shared(slot + i * word_bytes);
    if (inside(i)) {
      unpack<T>(v, f);
    } else {
      float e[N];
      unpack<T>(v, e);
#pragma unroll
      for (int k = 0; k < N; k += 2) f[k / 2] = make2(has(i, k) ? e[k] : 0.f, has(i, k + 1) ? e[k + 1] : 0.f);
    }
  }
  __device__ __forceinline__ void put(T* p, int i, const uint4& v) const {
    T* q = p + (tid * N - off) + i * (int)blockDim.x * N;
    if (inside(i)) {
      *reinterpret_cast<uint4*>(q) = v;
    } else {
      float e[N];
      unpack<T>(v, e);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (has(i, k)) Elem<T>::store1(q + k, e[k]);
    }
  }
  template <typename W>
  __device__ __forceinline__ void weight(const W* w, int i, F2* f) const {
    float e[N];
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = 0.f;
    if (live(i)) {
      if constexpr (!kShift) {
#pragma unroll
        for (int k = 0; k < N; k += Elem<W>::N) unpack<W>(__ldg(reinterpret_cast<const uint4*>(w + col(i, k))), e + k);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (has(i, k)) e[k] = Elem<W>::load1(w + col(i, k));
      }
    }
#pragma unroll
    for (int k = 0; k < N; k += 2) f[k / 2] = make2(e[k], e[k + 1]);
  }
};

// Sums over a row lane.  Warps leave their sums in `v`, whose entries behind the last warp hold zeros; turns alternate, so
// that a buffer is written again only when every thread has come past a barrier after reading it.
struct LaneSums {
  float v[2][kNormBarriers][kNormMaxWarps];
  __device__ __forceinline__ void clear(int tid, int lane, int warps) {
    if (warps > 1 && tid < kNormMaxWarps) v[0][lane][tid] = v[1][lane][tid] = 0.f;
    if (warps > 1) lane_barrier(1 + lane, blockDim.x);
  }
  __device__ __forceinline__ float total(int turn, int lane, int warps) const {
    float s = 0.f;
    for (int i = 0; i < warps; i += 4) {
      const float4 p = *reinterpret_cast<const float4*>(&v[turn][lane][i]);
      s += (p.x + p.y) + (p.z + p.w);
    }
    return s;
  }
};
__device__ __forceinline__ float part_sum(float v, int threads) {   // over a row lane of less than a warp
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  return threads == 8 ? v : v + __shfl_xor_sync(0xffffffffu, v, 8);
}
__device__ __forceinline__ float both(F2 v) {
  const float2 p = split2(v);
  return p.x + p.y;
}

template <typename T, typename W>
struct NormArgs {
  const T *x, *r;
  const W* w;
  T *y, *h;
  long long x_stride, r_stride, rows;
  int cols, stages;
  float eps;
};

template <typename T, typename W, int VPT, bool kShift>
__global__ void __launch_bounds__(kNormMaxThreads) add_rms_norm_kernel(const NormArgs<T, W> a) {
  constexpr int N = Elem<T>::N;
  extern __shared__ uint4 ring[];   // [stage][tensor][word][thread]
  __shared__ alignas(16) LaneSums sums;
  const RowLane<T, VPT, kShift> at(a.cols, ring);
  const bool sum = a.r != nullptr;
  const uint32_t tensor_bytes = VPT * at.word_bytes, stage_bytes = sum ? 2 * tensor_bytes : tensor_bytes;
  auto fetch = [&](long long row, uint32_t slot) {
    if (row < a.rows) {
      const long long left = kShift ? (a.rows - row) * a.cols : 0;
      at.fetch(slot, a.x + row * a.x_stride, left);
      if (sum) at.fetch(slot + tensor_bytes, a.r + row * a.r_stride, left);
    }
    copy_async_commit();
  };
  for (int s = 0; s + 1 < a.stages; ++s) fetch(at.row + s * at.step, at.ring + s * stage_bytes);
  F2 w[VPT][N / 2];
#pragma unroll
  for (int i = 0; i < VPT; ++i) at.weight(a.w, i, w[i]);
  sums.clear(at.tid, at.lane, at.warps);
  const float inv_cols = 1.f / (float)a.cols;
  uint32_t slot = at.ring, ahead = at.ring + (a.stages - 1) * stage_bytes;
  const uint32_t ring_end = at.ring + a.stages * stage_bytes;
  int turn = 0;
  long long row = at.row;
  for (long long wrow = at.warp_row; wrow < a.rows; wrow += at.step, row += at.step, turn ^= 1) {
    fetch(row + (a.stages - 1) * at.step, ahead);
    copy_async_wait(a.stages);
    const bool valid = row < a.rows;
    F2 v[VPT][N / 2], ss2 = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (valid && at.live(i)) {
        at.get(slot, i, v[i]);
        if (sum) {
          F2 q[N / 2];
          at.get(slot + tensor_bytes, i, q);
#pragma unroll
          for (int e = 0; e < N / 2; ++e) v[i][e] = add2(v[i][e], q[e]);
          const uint4 h = pack<T>(v[i]);
          at.put(a.h + row * a.cols, i, h);
          unpack<T>(h, v[i]);   // the norm is taken of what the stream holds
        }
#pragma unroll
        for (int e = 0; e < N / 2; ++e) ss2 = fma2(v[i][e], v[i][e], ss2);
      }
    }
    float ss = both(ss2);
    if (at.warps == 0) {
      ss = part_sum(ss, blockDim.x);
    } else {
      ss = warp_sum(ss);
      if (at.warps > 1) {
        if ((at.tid & 31) == 0) sums.v[turn][at.lane][at.tid >> 5] = ss;
        lane_barrier(1 + at.lane, blockDim.x);
        ss = sums.total(turn, at.lane, at.warps);
      }
    }
    const float rstd = rsqrtf(ss * inv_cols + a.eps);
    const F2 rstd2 = make2(rstd, rstd);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (valid && at.live(i)) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) v[i][e] = mul2(mul2(v[i][e], rstd2), w[i][e]);
        at.put(a.y + row * a.cols, i, pack<T>(v[i]));
      }
    }
    slot = slot + stage_bytes == ring_end ? at.ring : slot + stage_bytes;
    ahead = ahead + stage_bytes == ring_end ? at.ring : ahead + stage_bytes;
  }
}

template <typename T, typename W>
struct NormBwdArgs {
  const T *dy, *dh, *h;
  const W* w;
  T* dx;
  float* partial;   // (gridDim.x, cols): this CTA's part of dw, or nullptr
  long long dy_stride, dh_stride, h_stride, rows;
  int cols, stages;
  float eps;
};

// The row lanes of a CTA add their parts of dw in lane order through shared memory (the ring, once it is empty).
template <typename T, typename W, int VPT, bool kShift>
__global__ void __launch_bounds__(kNormMaxThreads) add_rms_norm_bwd_kernel(const NormBwdArgs<T, W> a) {
  constexpr int N = Elem<T>::N;
  extern __shared__ uint4 ring[];   // [stage][tensor][word][thread]
  __shared__ alignas(16) LaneSums square, cross;
  const RowLane<T, VPT, kShift> at(a.cols, ring);
  const bool stream = a.dh != nullptr;
  const uint32_t tensor_bytes = VPT * at.word_bytes, stage_bytes = (stream ? 3 : 2) * tensor_bytes;
  auto fetch = [&](long long row, uint32_t slot) {
    if (row < a.rows) {
      const long long left = kShift ? (a.rows - row) * a.cols : 0;
      at.fetch(slot, a.h + row * a.h_stride, left);
      at.fetch(slot + tensor_bytes, a.dy + row * a.dy_stride, left);
      if (stream) at.fetch(slot + 2 * tensor_bytes, a.dh + row * a.dh_stride, left);
    }
    copy_async_commit();
  };
  for (int s = 0; s + 1 < a.stages; ++s) fetch(at.row + s * at.step, at.ring + s * stage_bytes);
  F2 w[VPT][N / 2], dw[VPT][N / 2];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    at.weight(a.w, i, w[i]);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) dw[i][e] = 0;
  }
  square.clear(at.tid, at.lane, at.warps);
  cross.clear(at.tid, at.lane, at.warps);
  const float inv_cols = 1.f / (float)a.cols;
  uint32_t slot = at.ring, ahead = at.ring + (a.stages - 1) * stage_bytes;
  const uint32_t ring_end = at.ring + a.stages * stage_bytes;
  int turn = 0;
  long long row = at.row;
  for (long long wrow = at.warp_row; wrow < a.rows; wrow += at.step, row += at.step, turn ^= 1) {
    fetch(row + (a.stages - 1) * at.step, ahead);
    copy_async_wait(a.stages);
    const bool valid = row < a.rows;
    F2 ss2 = 0, sg2 = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (valid && at.live(i)) {
        F2 h[N / 2], dy[N / 2];
        at.get(slot, i, h);
        at.get(slot + tensor_bytes, i, dy);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          ss2 = fma2(h[e], h[e], ss2);
          sg2 = fma2(mul2(dy[e], w[i][e]), h[e], sg2);
        }
      }
    }
    float ss = both(ss2), sg = both(sg2);
    if (at.warps == 0) {
      ss = part_sum(ss, blockDim.x);
      sg = part_sum(sg, blockDim.x);
    } else {
      ss = warp_sum(ss);
      sg = warp_sum(sg);
      if (at.warps > 1) {
        if ((at.tid & 31) == 0) {
          square.v[turn][at.lane][at.tid >> 5] = ss;
          cross.v[turn][at.lane][at.tid >> 5] = sg;
        }
        lane_barrier(1 + at.lane, blockDim.x);
        ss = square.total(turn, at.lane, at.warps);
        sg = cross.total(turn, at.lane, at.warps);
      }
    }
    const float rstd = rsqrtf(ss * inv_cols + a.eps);
    const float mean_gn = sg * rstd * inv_cols;
    const F2 rstd2 = make2(rstd, rstd), back = make2(-mean_gn, -mean_gn);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (valid && at.live(i)) {
        F2 h[N / 2], dy[N / 2], o[N / 2];
        at.get(slot, i, h);
        at.get(slot + tensor_bytes, i, dy);
        if (stream) {
          at.get(slot + 2 * tensor_bytes, i, o);
        } else {
#pragma unroll
          for (int e = 0; e < N / 2; ++e) o[e] = 0;
        }
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const F2 n = mul2(h[e], rstd2);
          dw[i][e] = fma2(dy[e], n, dw[i][e]);
          o[e] = fma2(rstd2, fma2(n, back, mul2(dy[e], w[i][e])), o[e]);
        }
        at.put(a.dx + row * a.cols, i, pack<T>(o));
      }
    }
    slot = slot + stage_bytes == ring_end ? at.ring : slot + stage_bytes;
    ahead = ahead + stage_bytes == ring_end ? at.ring : ahead + stage_bytes;
  }
  if (a.partial == nullptr) return;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // every thread is through with its part of the ring
  float* dw_part = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (at.live(i)) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 p = split2(dw[i][e / 2]);
        if (at.has(i, e)) dw_part[at.lane * a.cols + at.col(i, e)] = e % 2 ? p.y : p.x;
      }
    }
  }
  __syncthreads();
  for (int col = threadIdx.y * blockDim.x + threadIdx.x; col < a.cols; col += blockDim.x * blockDim.y) {
    float s = dw_part[col];
    for (int l = 1; l < blockDim.y; ++l) s += dw_part[l * a.cols + col];
    a.partial[(long long)blockIdx.x * a.cols + col] = s;
  }
}

// dw[c] = sum over the CTAs' parts, in a fixed order: 32 columns a CTA, 32 parts at a time.  Launched while the kernel above
// runs out (programmatic dependent launch): it waits for that kernel's end where it stands.
template <typename W>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* partial, W* __restrict__ dw, int parts, int cols) {
  __shared__ float s[32][33];
  const int x = threadIdx.x, y = threadIdx.y, c = blockIdx.x * 32 + x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float acc = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int p = y; p < parts; p += 32) acc += partial[(long long)p * cols + c];
  }
  s[y][x] = acc;
  __syncthreads();
  acc = warp_sum(s[x][y]);
  if (x == 0 && blockIdx.x * 32 + y < cols) Elem<W>::store1(dw + blockIdx.x * 32 + y, acc);
}

}  // namespace b200train
