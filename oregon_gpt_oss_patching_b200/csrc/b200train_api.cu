// C ABI of the training-step entry points (declared in include/b200train.h): argument validation and kernel launches.
// No device memory is allocated here and nothing synchronises.
#include "../../include/b200train.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <memory>
#include <new>
#include <utility>

#include "clip_kernels.cuh"
#include "host_common.cuh"
#include "norm_kernels.cuh"

namespace {

using namespace b200train;
using namespace b200attn::host;

// (asked for several times a call: looked up once a device)
int sm_count(int device) {
  static std::atomic<int> known[kMaxDevices];
  const bool cacheable = device >= 0 && device < kMaxDevices;
  int n = cacheable ? known[device].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) return 148;
  if (cacheable) known[device].store(n, std::memory_order_relaxed);
  return n;
}

int elem_size(int dtype) { return dtype == B200TRAIN_FP32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype >= B200TRAIN_BF16 && dtype <= B200TRAIN_FP32; }

// Launches a kernel that may start while the one before it in the stream runs out; it waits for that one's end itself.
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), unsigned grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  const bool launched = cudaLaunchKernelEx(&config, kernel, args...) == cudaSuccess;
  return launch_status() == B200ATTN_OK && launched ? B200ATTN_OK : B200ATTN_ECUDA;   // (the error is taken off the thread, as after <<<>>>)
}

// ---------------------------------------------------------------- norm

// Elements a thread holds: the instances of the two kernels, the preferred ones first (16-bit and 32-bit types).
constexpr int kNormElems16[] = {24, 32, 16, 8}, kNormElems32[] = {16, 24, 32, 8};
constexpr size_t kNormSmem = 216 * 1024;        // of a CTA's ring (static shared memory comes on top)

struct NormShape {
  int elems = 0;     // one of kNormElems, 0: the row is too wide
  int threads = 0;   // of a row lane
  int lanes = 0;     // row lanes of a CTA
  int grid = 0;
  int stages = 0;    // of the ring
  size_t smem = 0;
  bool shift = false;
};

// The piece of a row a thread that leaves the fewest threads without a word of it; where there are not rows enough for every
// SM, the one that spreads a row over the most threads.  Then as many row lanes as there are threads and rows for, a ring of
// three rows a lane where shared memory holds that for all of them, and of two otherwise.
NormShape norm_shape(long long rows, int cols, int dtype, int device, int tensors) {
  NormShape s;
  const int n = 16 / elem_size(dtype), sms = sm_count(device);
  s.shift = cols % n != 0;
  const int words = (cols + n - 1) / n + (s.shift ? 1 : 0);
  const bool few = rows <= sms;
  long long held = 0;   // words that the threads of a row lane have room for
  for (int e : dtype == B200TRAIN_FP32 ? kNormElems32 : kNormElems16) {
    const int per_thread = e / n;
    int threads = (words + per_thread - 1) / per_thread;
    threads = threads <= 8 ? 8 : threads <= 16 ? 16 : (threads + 31) / 32 * 32;
    if (threads > kNormMaxThreads) continue;
    if (s.elems != 0 && (few ? threads <= s.threads : (long long)threads * per_thread >= held)) continue;
    s.elems = e;
    s.threads = threads;
    held = (long long)threads * per_thread;
  }
  if (s.elems == 0) return s;
  const size_t lane_stage = (size_t)s.threads * (s.elems / n) * 16 * tensors;   // bytes of one row of the ring
  const size_t all = lane_stage * (kNormMaxThreads / s.threads);                 // of one row of every lane that has threads
  s.stages = all * 3 <= kNormSmem ? 3 : lane_stage * 2 <= kNormSmem ? 2 : 1;
  const int unit = s.threads < 32 ? 32 / s.threads : 1;   // lanes come in whole warps
  int most = std::min((int)(kNormSmem / (lane_stage * s.stages)), kNormMaxThreads / s.threads);
  if (s.threads > 32) most = std::min(most, kNormBarriers);
  const long long spread = std::max(1ll, (rows + sms - 1) / sms);   // rows an SM
  const int lanes = (int)std::min<long long>(most / unit * unit, (spread + unit - 1) / unit * unit);
  s.lanes = lanes;
  s.smem = lane_stage * s.stages * lanes;
  const long long want = std::max(1ll, (rows + lanes - 1) / lanes);
  s.grid = (int)std::min<long long>(want, sms);
  if (s.shift && want > s.grid) {   // a lane's rows step by a multiple of 8 (see the kernels)
    while (s.grid * lanes % 8 != 0 && s.grid > 1) --s.grid;
    if (s.grid * lanes % 8 != 0) s.grid = 8;
  }
  return s;
}

int check_norm_matrix(const void* p, int64_t stride, int64_t rows, int cols, int dtype) {
  if (rows == 0) return B200ATTN_OK;   // (an empty tensor has no address)
  if (p == nullptr) return B200ATTN_EINVAL;
  const int n = 16 / elem_size(dtype);
  if (!aligned16(p) || stride < 0) return B200ATTN_EALIGN;
  if (cols % n == 0 ? stride % n != 0 : stride != cols) return B200ATTN_EALIGN;
  return B200ATTN_OK;
}

int check_norm(int64_t rows, int cols, int dtype, int weight_dtype, const void* weight, float eps) {
  if (rows < 0 || cols <= 0 || weight == nullptr || !known_dtype(dtype) || !(eps >= 0.f)) return B200ATTN_EINVAL;
  if (weight_dtype != dtype && weight_dtype != B200TRAIN_FP32) return B200ATTN_EINVAL;
  if (cols > B200TRAIN_NORM_MAX_COLS || rows > (1ll << 40) / cols) return B200ATTN_ESHAPE;
  return aligned16(weight) ? B200ATTN_OK : B200ATTN_EALIGN;
}

// Calls f(T{}, W{}) with the element type and the weight type.
template <typename F>
int with_types(int dtype, int weight_dtype, F f) {
  if (dtype == B200TRAIN_FP32) return f(float{}, float{});
  if (dtype == B200TRAIN_BF16) return weight_dtype == B200TRAIN_FP32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
  return weight_dtype == B200TRAIN_FP32 ? f(__half{}, float{}) : f(__half{}, __half{});
}

// Calls f(integral_constant<int, words a thread holds>, bool_constant<shift>).
template <int V>
struct Int {
  static constexpr int value = V;
};
template <int N, typename F>
int with_shape(const NormShape& s, F f) {
  switch (s.elems) {
    case 8: return s.shift ? f(Int<8 / N>{}, Int<1>{}) : f(Int<8 / N>{}, Int<0>{});
    case 16: return s.shift ? f(Int<16 / N>{}, Int<1>{}) : f(Int<16 / N>{}, Int<0>{});
    case 24: return s.shift ? f(Int<24 / N>{}, Int<1>{}) : f(Int<24 / N>{}, Int<0>{});
    default: return s.shift ? f(Int<32 / N>{}, Int<1>{}) : f(Int<32 / N>{}, Int<0>{});
  }
}

// ---------------------------------------------------------------- clip

// CTAs an SM: of 3, 4, 6 and 8 the fastest on one decoder layer's gradients (within 4 % of one another).
constexpr int kSumCtas = 6, kApplyCtas = 4;
// Shared memory that the second kernel takes and does not use: no SM has room for a fifth CTA.  They arrive while the first
// kernel runs out, and would crowd on the SMs that are free first (clip 882 us instead of 780).
constexpr size_t kApplySmem = 46 * 1024;

enum class ClipOp { kNorm, kClip, kSgd };

// Fills a table with the tensors [begin, begin + kClipTensors), empty ones left out, and returns how many were looked at.
int64_t fill_table(ClipTable* t, const int64_t* grads, const int64_t* params, const int64_t* counts, const int32_t* dtypes, int64_t begin,
                   int64_t tensors) {
  t->tensors = 0;
  unsigned chunks = 0;
  int64_t i = begin;
  for (; i < tensors && t->tensors < kClipTensors; ++i) {
    if (counts[i] == 0) continue;
    const long long n = 16 / elem_size(dtypes[i]);
    const long long off = (long long)(((uint64_t)grads[i] & 15u) / elem_size(dtypes[i]));
    const int k = t->tensors++;
    t->grad[k] = reinterpret_cast<void*>((uintptr_t)grads[i]);
    t->param[k] = params != nullptr ? reinterpret_cast<void*>((uintptr_t)params[i]) : nullptr;
    t->count[k] = counts[i];
    t->first[k] = chunks;
    t->dtype[k] = (unsigned char)dtypes[i];
    chunks += (unsigned)(((off + counts[i] + n - 1) / n + kChunkWords - 1) / kChunkWords);
  }
  t->chunks = chunks;
  return i - begin;
}

// Whether any two of the tensors that are written share memory, with one another or with a tensor that is read.
bool overlaps(const int64_t* a, const int64_t* b, const int64_t* counts, const int32_t* dtypes, int64_t n) {
  std::pair<uint64_t, uint64_t> few[128];
  std::unique_ptr<std::pair<uint64_t, uint64_t>[]> many;
  const int64_t all = b != nullptr ? 2 * n : n;
  auto* s = few;
  if (all > 128) {
    many.reset(new (std::nothrow) std::pair<uint64_t, uint64_t>[all]);
    if (!many) return true;
    s = many.get();
  }
  int64_t k = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    const uint64_t bytes = (uint64_t)counts[i] * elem_size(dtypes[i]);
    s[k++] = {(uint64_t)a[i], (uint64_t)a[i] + bytes};
    if (b != nullptr) s[k++] = {(uint64_t)b[i], (uint64_t)b[i] + bytes};
  }
  std::sort(s, s + k);
  for (int64_t i = 1; i < k; ++i)
    if (s[i].first < s[i - 1].second) return true;
  return false;
}

int run_clip(ClipOp op, const int64_t* grads, const int64_t* params, const int64_t* counts, const int32_t* dtypes, int64_t tensors, float lr,
             float max_norm, double* scratch, int64_t scratch_doubles, float* norm, int device, void* stream) {
  if (tensors < 0 || norm == nullptr || (tensors > 0 && (grads == nullptr || counts == nullptr || dtypes == nullptr))) return B200ATTN_EINVAL;
  if (op == ClipOp::kSgd && tensors > 0 && params == nullptr) return B200ATTN_EINVAL;
  if (op != ClipOp::kNorm && !(max_norm >= 0.f)) return B200ATTN_EINVAL;
  if (tensors > (1 << 24)) return B200ATTN_ESHAPE;
  int64_t left = 1ll << 43;   // elements in all: at most 2^30 chunks, and one more a tensor, fit the 32 bits of a chunk's number
  for (int64_t i = 0; i < tensors; ++i) {
    if (!known_dtype(dtypes[i]) || counts[i] < 0) return B200ATTN_EINVAL;
    if (counts[i] > left) return B200ATTN_ESHAPE;
    left -= counts[i];
    if (counts[i] == 0) continue;
    const int64_t size = elem_size(dtypes[i]);
    if (grads[i] == 0 || (op == ClipOp::kSgd && params[i] == 0)) return B200ATTN_EINVAL;
    if (grads[i] % size != 0 || (op == ClipOp::kSgd && params[i] % size != 0)) return B200ATTN_EALIGN;
  }
  if (op != ClipOp::kNorm && overlaps(grads, op == ClipOp::kSgd ? params : nullptr, counts, dtypes, tensors)) return B200TRAIN_EOVERLAP;
  int rc = check_device(device);
  if (rc) return rc;
  if (scratch == nullptr || scratch_doubles < b200train_clip_scratch_doubles(tensors, device)) return B200ATTN_ESCRATCH;
  DeviceGuard guard(device);
  if (!guard.ok) return B200ATTN_ECUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(device);
  ClipTable t;
  int parts = 0;
  for (int64_t i = 0; i < tensors;) {
    i += fill_table(&t, grads, params, counts, dtypes, i, tensors);
    if (t.tensors == 0) continue;
    const int grid = (int)std::min<unsigned>(t.chunks, sms * kSumCtas);
    grad_sumsq_kernel<<<grid, kClipThreads, 0, st>>>(t, scratch + parts);
    parts += grid;
    if ((rc = launch_status())) return rc;
  }
  const double* partials = scratch;
  if (op == ClipOp::kNorm || parts == 0) return launch_dependent(grad_norm_kernel, 1, dim3(kClipThreads), 0, st, partials, parts, norm);
  auto* apply = op == ClipOp::kSgd ? clip_apply_kernel<true> : clip_apply_kernel<false>;
  for (int64_t i = 0; i < tensors;) {
    if (tensors > kClipTensors) i += fill_table(&t, grads, params, counts, dtypes, i, tensors);
    else i = tensors;   // (the table of the first kernel serves again)
    if (t.tensors == 0) continue;
    rc = launch_dependent(apply, std::min<unsigned>(t.chunks, sms * kApplyCtas), dim3(kClipThreads), kApplySmem, st, t, partials, parts, max_norm,
                          lr, norm);
    if (rc) return rc;
  }
  return B200ATTN_OK;
}

}  // namespace

extern "C" {

int b200train_add_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                           const void* weight, void* y, void* h, int64_t rows, int32_t cols, float eps, int32_t dtype,
                           int32_t weight_dtype, int32_t device, void* stream) {
  int rc = check_norm(rows, cols, dtype, weight_dtype, weight, eps);
  if (rc) return rc;
  if (rows > 0 && (residual == nullptr) != (h == nullptr)) return B200ATTN_EINVAL;
  if ((rc = check_norm_matrix(x, x_stride, rows, cols, dtype)) || (rc = check_norm_matrix(y, cols, rows, cols, dtype))) return rc;
  if (residual != nullptr &&
      ((rc = check_norm_matrix(residual, residual_stride, rows, cols, dtype)) || (rc = check_norm_matrix(h, cols, rows, cols, dtype))))
    return rc;
  if ((rc = check_device(device))) return rc;
  const NormShape s = norm_shape(rows, cols, dtype, device, residual != nullptr ? 2 : 1);
  if (s.elems == 0) return B200ATTN_ESHAPE;
  if (rows == 0) return B200ATTN_OK;
  DeviceGuard guard(device);
  if (!guard.ok) return B200ATTN_ECUDA;
  return with_types(dtype, weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    NormArgs<T, W> a{static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const W*>(weight), static_cast<T*>(y),
                     static_cast<T*>(h), x_stride, residual_stride, rows, cols, s.stages, eps};
    return with_shape<Elem<T>::N>(s, [&](auto vpt, auto shift) {
      constexpr auto kernel = add_rms_norm_kernel<T, W, decltype(vpt)::value, decltype(shift)::value != 0>;
      if (int e = set_smem<kernel>(kNormSmem)) return e;
      kernel<<<s.grid, dim3(s.threads, s.lanes), s.smem, static_cast<cudaStream_t>(stream)>>>(a);
      return launch_status();
    });
  });
}

int64_t b200train_norm_scratch_floats(int64_t rows, int32_t cols, int32_t dtype, int32_t device) {
  if (rows <= 0 || cols <= 0 || cols > B200TRAIN_NORM_MAX_COLS || !known_dtype(dtype)) return 0;
  // (a pass without dh may take more row lanes a CTA, never more CTAs than there are SMs)
  return (int64_t)std::min<int64_t>(rows, std::max(sm_count(device), 8)) * cols;
}

int b200train_add_rms_norm_bwd(const void* dy, int64_t dy_stride, const void* dh, int64_t dh_stride, const void* h,
                               int64_t h_stride, const void* weight, void* dx, void* dweight, float* scratch,
                               int64_t scratch_floats, int64_t rows, int32_t cols, float eps, int32_t dtype,
                               int32_t weight_dtype, int32_t device, void* stream) {
  int rc = check_norm(rows, cols, dtype, weight_dtype, weight, eps);
  if (rc) return rc;
  if ((rc = check_norm_matrix(dy, dy_stride, rows, cols, dtype)) || (rc = check_norm_matrix(h, h_stride, rows, cols, dtype)) ||
      (rc = check_norm_matrix(dx, cols, rows, cols, dtype)))
    return rc;
  if (dh != nullptr && (rc = check_norm_matrix(dh, dh_stride, rows, cols, dtype))) return rc;
  if ((rc = check_device(device))) return rc;
  const NormShape s = norm_shape(rows, cols, dtype, device, dh != nullptr ? 3 : 2);
  if (s.elems == 0) return B200ATTN_ESHAPE;
  DeviceGuard guard(device);
  if (!guard.ok) return B200ATTN_ECUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return dweight == nullptr || cudaMemsetAsync(dweight, 0, (size_t)cols * elem_size(weight_dtype), st) == cudaSuccess ? B200ATTN_OK
                                                                                                                         : B200ATTN_ECUDA;
  if (dweight != nullptr && (scratch == nullptr || scratch_floats < (int64_t)s.grid * cols)) return B200ATTN_ESCRATCH;
  return with_types(dtype, weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    NormBwdArgs<T, W> a{static_cast<const T*>(dy), static_cast<const T*>(dh), static_cast<const T*>(h), static_cast<const W*>(weight),
                        static_cast<T*>(dx), dweight != nullptr ? scratch : nullptr, dy_stride, dh_stride, h_stride, rows, cols, s.stages, eps};
    int rc2 = with_shape<Elem<T>::N>(s, [&](auto vpt, auto shift) {
      constexpr auto kernel = add_rms_norm_bwd_kernel<T, W, decltype(vpt)::value, decltype(shift)::value != 0>;
      if (int e = set_smem<kernel>(kNormSmem)) return e;
      kernel<<<s.grid, dim3(s.threads, s.lanes), s.smem, st>>>(a);
      return launch_status();
    });
    if (rc2 || dweight == nullptr) return rc2;
    return launch_dependent(norm_dw_kernel<W>, (cols + 31) / 32, dim3(32, 32), 0, st, static_cast<const float*>(scratch), static_cast<W*>(dweight),
                            s.grid, cols);
  });
}

// (one partial a CTA of every launch; every launch but the last takes kClipTensors tensors)
int64_t b200train_clip_scratch_doubles(int64_t tensors, int32_t device) {
  if (tensors < 0) return 0;
  return (tensors / kClipTensors + 1) * sm_count(device) * kSumCtas;
}

int b200train_grad_norm(const int64_t* grads, const int64_t* counts, const int32_t* dtypes, int64_t tensors, double* scratch,
                        int64_t scratch_doubles, float* norm, int32_t device, void* stream) {
  return run_clip(ClipOp::kNorm, grads, nullptr, counts, dtypes, tensors, 0.f, 0.f, scratch, scratch_doubles, norm, device, stream);
}

int b200train_clip_grads(const int64_t* grads, const int64_t* counts, const int32_t* dtypes, int64_t tensors, float max_norm,
                         double* scratch, int64_t scratch_doubles, float* norm, int32_t device, void* stream) {
  return run_clip(ClipOp::kClip, grads, nullptr, counts, dtypes, tensors, 0.f, max_norm, scratch, scratch_doubles, norm, device, stream);
}

int b200train_clipped_sgd(const int64_t* grads, const int64_t* params, const int64_t* counts, const int32_t* dtypes, int64_t tensors,
                          float lr, float max_norm, double* scratch, int64_t scratch_doubles, float* norm, int32_t device, void* stream) {
  return run_clip(ClipOp::kSgd, grads, params, counts, dtypes, tensors, lr, max_norm, scratch, scratch_doubles, norm, device, stream);
}

}  // extern "C"
