// The training-step operators as torch functions: argument checks, allocations and autograd around the C ABI of
// include/b200train.h and the router of include/b200moe.h.  Host code alone, one extension module.
//
// The attention and expert wrappers do this in Python; these operators are called once or twice a layer on little data (or on
// hundreds of small tensors), where the host's time is what a caller waits for: a norm of a few rows takes 7.5 us of it here and 14 us
// through Python and ctypes, a forward with its backward 55 us and 94 us (40 us of them autograd's own), the routing of a few
// tokens 6 us and 22 us, clipping 48 gradients 18 us and 50 us.
//
// The module calls the library through addresses it is given (set_library), so that there is one loaded copy of it, the one
// that the Python side found, checked and reports on.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <limits>
#include <optional>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/b200moe.h"
#include "../../include/b200train.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Library {
  decltype(&b200attn_strerror) strerror = nullptr;
  decltype(&b200train_add_rms_norm) add_rms_norm = nullptr;
  decltype(&b200train_norm_scratch_floats) norm_scratch_floats = nullptr;
  decltype(&b200train_add_rms_norm_bwd) add_rms_norm_bwd = nullptr;
  decltype(&b200train_clip_scratch_doubles) clip_scratch_doubles = nullptr;
  decltype(&b200train_grad_norm) grad_norm = nullptr;
  decltype(&b200train_clip_grads) clip_grads = nullptr;
  decltype(&b200train_clipped_sgd) clipped_sgd = nullptr;
  decltype(&b200moe_router_topk) router_topk = nullptr;
  decltype(&b200moe_router_topk_bwd) router_topk_bwd = nullptr;
} lib;

template <typename F>
void take_address(F& f, const std::unordered_map<std::string, uintptr_t>& addresses, const char* name) {
  const auto at = addresses.find(name);
  TORCH_CHECK(at != addresses.end() && at->second != 0, "libb200attn.so has no ", name);
  f = reinterpret_cast<F>(at->second);
}

void set_library(const std::unordered_map<std::string, uintptr_t>& a) {
  take_address(lib.strerror, a, "b200attn_strerror");
  take_address(lib.add_rms_norm, a, "b200train_add_rms_norm");
  take_address(lib.norm_scratch_floats, a, "b200train_norm_scratch_floats");
  take_address(lib.add_rms_norm_bwd, a, "b200train_add_rms_norm_bwd");
  take_address(lib.clip_scratch_doubles, a, "b200train_clip_scratch_doubles");
  take_address(lib.grad_norm, a, "b200train_grad_norm");
  take_address(lib.clip_grads, a, "b200train_clip_grads");
  take_address(lib.clipped_sgd, a, "b200train_clipped_sgd");
  take_address(lib.router_topk, a, "b200moe_router_topk");
  take_address(lib.router_topk_bwd, a, "b200moe_router_topk_bwd");
}

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed: ", lib.strerror(rc), " (code ", rc, ")"); }

// Forward-mode derivatives would be lost here without a word: nothing below looks at a tangent.
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool has_tangent(const std::optional<Tensor>& t) { return t.has_value() && has_tangent(*t); }
template <typename... T>
void check_no_tangent(const char* name, const T&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(tensors) || ...), name, " has no forward-mode derivative");
}
// A trace would keep this call's results as constants.
void check_not_traced(const char* name) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), name, " cannot be traced: the trace would keep its results for these inputs");
}
// Whether any tensor can have a tangent: asked once where there are many of them.
bool tangents_exist() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

// B200TRAIN_* and B200MOE_* (the same numbers), -1 for any other type
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return B200TRAIN_BF16;
    case at::kHalf: return B200TRAIN_FP16;
    case at::kFloat: return B200TRAIN_FP32;
    default: return -1;
  }
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }
// A tensor's address.  Fake tensors and wrappers of others pass for CUDA tensors and have no memory of their own; an offset into
// nothing would be an address like any other.
const void* address(const Tensor& t) {
  TORCH_CHECK(t.numel() == 0 || t.storage().data() != nullptr, "needs tensors with memory of their own, got one without (a fake tensor or a wrapper)");
  return t.const_data_ptr();
}
template <typename... T>
void check_memory(const T&... tensors) {
  const auto look = [](const std::optional<Tensor>& t) {
    if (t.has_value()) address(*t);
  };
  (look(tensors), ...);
}
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(address(t)) % 16 == 0; }
// A tensor whose memory holds its values: the imaginary part of a conjugate, for one, is a view that torch negates where it reads it.
Tensor as_it_lies(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor copy_of(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
// A contiguous tensor on x's device, without the dispatcher's way there (half the time of at::empty, and most calls make two to five).
Tensor empty_on(const Tensor& x, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, x.device(), std::nullopt);
}
const void* data(const Tensor& t) { return t.defined() ? address(t) : nullptr; }

// ---------------------------------------------------------------- norm

// Rows that the kernels can address in place (`t` itself or a view of it), or a contiguous copy, with the row stride.
struct Rows {
  Tensor t;
  int64_t stride;
  Rows() : stride(0) {}
  Rows(const Tensor& of, int64_t cols) : t(as_it_lies(of)), stride(cols) {
    if (!t.is_contiguous()) {
      t = t.reshape({-1, cols});
      const int64_t per_word = 16 / static_cast<int64_t>(t.element_size());
      if (!t.is_contiguous()) {
        if (t.stride(1) != 1 || cols % per_word != 0 || t.stride(0) % per_word != 0) t = t.contiguous();
        else stride = t.stride(0);
      }
    }
    if (!aligned16(t)) {
      t = copy_of(t);
      stride = cols;
    }
  }
};

void check_norm(const char* name, const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps) {
  TORCH_CHECK(x.is_cuda(), name, " needs CUDA tensors (the sm_100a library is the only code path)");
  TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0, name, " supports bfloat16, float16 and float32, got ", x.dtype());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, name, ": x must have a last dimension to normalise, got shape ", x.sizes());
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), name, ": weight must be (", x.size(-1), ",), got ", weight.sizes());
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, name, ": weight must be ", x.dtype(),
                   " or float32, got ", weight.dtype());
  TORCH_CHECK(weight.device() == x.device(), name, ": weight is on ", weight.device(), ", x on ", x.device());
  if (residual.has_value())
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device(), name,
                      ": residual must match x (", x.sizes(), ", ", x.dtype(), ", ", x.device(), "), got ", residual->sizes(), ", ",
                      residual->dtype(), ", ", residual->device());
  TORCH_CHECK_VALUE(eps >= 0.0, name, ": eps must not be negative, got ", eps);
  TORCH_CHECK_VALUE(x.size(-1) <= std::numeric_limits<int32_t>::max(), name, ": rows of ", x.size(-1), " elements");
  check_not_traced(name);
  check_memory(x, residual, weight);
  check_no_tangent(name, x, residual, weight);
}

// A weight as the kernels read it: contiguous, on the 16-byte grid.
Tensor on_grid(const Tensor& w) { return w.is_contiguous() && !w.is_neg() && aligned16(w) ? w : copy_of(w); }

// A saved value that comes back through a hook (an offload, a compression) may lie otherwise in memory than it did: each is laid
// out for the kernels again, once it is known to be what was saved.
void check_saved(const char* name, const Tensor& saved, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
  TORCH_CHECK(saved.sizes() == sizes && saved.scalar_type() == type && saved.device() == device, name, ": a saved tensor came back as ",
              saved.sizes(), ", ", saved.dtype(), ", ", saved.device(), "; saved were ", sizes, ", ", type, ", ", device);
}

struct Normed {
  Tensor y, h;      // h undefined without a residual
  Tensor kept;      // what the backward reads as h
  Tensor weight;
};

Normed norm_forward(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps) {
  const int64_t cols = x.size(-1);
  const int device = x.get_device();
  Normed n;
  const Rows in(x, cols);
  n.weight = on_grid(weight);
  n.y = empty_on(x, x.sizes(), x.scalar_type());
  Rows r;
  if (residual.has_value()) {
    r = Rows(*residual, cols);
    n.h = empty_on(x, x.sizes(), x.scalar_type());
    n.kept = n.h;
  } else {
    n.kept = in.t;
  }
  check(lib.add_rms_norm(data(in.t), in.stride, data(r.t), r.stride, data(n.weight), n.y.mutable_data_ptr(),
                         n.h.defined() ? n.h.mutable_data_ptr() : nullptr, x.numel() / cols, static_cast<int32_t>(cols),
                         static_cast<float>(eps), dtype_code(x.scalar_type()), dtype_code(n.weight.scalar_type()), device, stream_of(device)),
        "b200train_add_rms_norm");
  return n;
}

// A node of torch's graph, built here rather than through torch::autograd::Function: its saved values are members instead of a
// dictionary, which takes 9 us off a forward and its backward.
template <typename N>
std::shared_ptr<N> new_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

struct AddRmsNormBackward : Node {
  SavedVariable h, weight;
  std::vector<int64_t> saved_sizes;   // of h
  at::ScalarType weight_type = at::kFloat;
  double eps = 0.0;
  std::string name() const override { return "AddRmsNormBackward"; }
  void release_variables() override {
    h.reset_data();
    weight.reset_data();
  }
  // (dy, dh) -> (dx, dresidual, dweight)
  variable_list apply(variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(), "add_rms_norm cannot be differentiated twice");
    const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    const Tensor none;
    const bool residual = task_should_compute_output(1);
    if (!dy.defined()) return {dh, residual ? dh : none, none};   // the norm was not used: the stream's gradient passes through
    const int64_t cols = dy.size(-1), rows = dy.numel() / cols;
    const int device = dy.get_device(), dtype = dtype_code(dy.scalar_type());
    const Tensor saved = h.unpack(shared_from_this()), saved_weight = weight.unpack();
    check_saved("add_rms_norm", saved, saved_sizes, dy.scalar_type(), dy.device());
    check_saved("add_rms_norm", saved_weight, {cols}, weight_type, dy.device());
    const Tensor w = on_grid(saved_weight);
    const Rows hs(saved, cols), dyr(dy, cols), dhr = dh.defined() ? Rows(dh, cols) : Rows();
    Tensor dx = empty_on(dy, dy.sizes(), dy.scalar_type()), dw, scratch;
    int64_t floats = 0;
    if (task_should_compute_output(2)) {
      dw = empty_on(w, w.sizes(), w.scalar_type());
      floats = lib.norm_scratch_floats(rows, static_cast<int32_t>(cols), dtype, device);
      scratch = empty_on(dy, {floats}, at::kFloat);
    }
    check(lib.add_rms_norm_bwd(data(dyr.t), dyr.stride, data(dhr.t), dhr.stride, data(hs.t), hs.stride, data(w), dx.mutable_data_ptr(),
                               dw.defined() ? dw.mutable_data_ptr() : nullptr, scratch.defined() ? scratch.mutable_data_ptr<float>() : nullptr,
                               floats, rows, static_cast<int32_t>(cols), static_cast<float>(eps), dtype, dtype_code(w.scalar_type()), device,
                               stream_of(device)),
          "b200train_add_rms_norm_bwd");
    return {dx, residual ? dx : none, dw};
  }
};

// (y, h) with their history: h is the sum; without a residual x itself if `passed`, undefined otherwise.
std::pair<Tensor, Tensor> differentiable_norm(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps, bool passed) {
  Normed n;
  Tensor h;
  {
    at::NoGradGuard no_grad;
    n = norm_forward(x, residual, weight, eps);
    h = residual.has_value() || !passed ? n.h : x.detach();   // (the stream's own memory and version, with a history of its own)
  }
  auto node = new_node<AddRmsNormBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x, residual.has_value() ? *residual : Tensor(), weight));
  node->saved_sizes = n.kept.sizes().vec();
  node->weight_type = n.weight.scalar_type();
  node->eps = eps;
  torch::autograd::set_history(n.y, node);
  if (h.defined()) torch::autograd::set_history(h, node);
  node->h = residual.has_value() ? SavedVariable(h, true) : SavedVariable(n.kept, false);
  node->weight = SavedVariable(n.weight, false);
  return {n.y, h};
}

bool differentiates(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight) {
  return at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (residual.has_value() && residual->requires_grad()));
}

std::pair<Tensor, Tensor> add_rms_norm(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps) {
  check_norm("add_rms_norm", x, residual, weight, eps);
  if (differentiates(x, residual, weight)) return differentiable_norm(x, residual, weight, eps, true);
  Normed n = norm_forward(x, residual, weight, eps);
  return {n.y, n.h.defined() ? n.h : x};
}

Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps) {
  check_norm("rms_norm", x, std::nullopt, weight, eps);
  if (differentiates(x, std::nullopt, weight)) return differentiable_norm(x, std::nullopt, weight, eps, false).first;
  return norm_forward(x, std::nullopt, weight, eps).y;
}

// ---------------------------------------------------------------- router

struct Routing {
  int64_t top_k, num_groups, top_groups;
  bool sigmoid, renormalize;
  double scale;
};

std::pair<Tensor, Tensor> router_forward(const Tensor& logits, const std::optional<Tensor>& bias, const Routing& how) {
  const int device = logits.get_device();
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  Tensor b;
  if (bias.has_value()) b = as_it_lies(bias->to(at::kFloat)).contiguous();
  Tensor weights = empty_on(logits, {tokens, how.top_k}, logits.scalar_type());
  Tensor indices = empty_on(logits, {tokens, how.top_k}, at::kLong);
  check(lib.router_topk(data(logits), logits.stride(0), static_cast<const float*>(data(b)), weights.mutable_data_ptr(),
                        indices.mutable_data_ptr<int64_t>(), static_cast<int32_t>(tokens), static_cast<int32_t>(experts),
                        static_cast<int32_t>(how.top_k), static_cast<int32_t>(how.num_groups), static_cast<int32_t>(how.top_groups), how.sigmoid,
                        how.renormalize, static_cast<float>(how.scale), dtype_code(logits.scalar_type()), device, stream_of(device)),
        "b200moe_router_topk");
  return {weights, indices};
}

// A row's elements lie next to each other.
Tensor row_major(const Tensor& logits) {
  const Tensor l = as_it_lies(logits);
  return l.stride(1) == 1 || l.size(1) == 1 ? l : l.contiguous();
}

struct RouterTopkBackward : Node {
  SavedVariable logits, indices;
  int64_t experts = 0;
  bool sigmoid = false, renormalize = false;
  double scale = 1.0;
  std::string name() const override { return "RouterTopkBackward"; }
  void release_variables() override {
    logits.reset_data();
    indices.reset_data();
  }
  // (dweights) -> (dlogits)
  variable_list apply(variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(), "router_topk cannot be differentiated twice");
    if (!grads[0].defined()) return {Tensor()};
    const Tensor dweights = as_it_lies(grads[0]).contiguous(), saved = logits.unpack(), saved_indices = indices.unpack();
    check_saved("router_topk", saved, {dweights.size(0), experts}, dweights.scalar_type(), dweights.device());
    check_saved("router_topk", saved_indices, dweights.sizes(), at::kLong, dweights.device());
    const Tensor l = row_major(saved), chosen = saved_indices.contiguous();
    const int device = l.get_device();
    Tensor dlogits = empty_on(l, l.sizes(), l.scalar_type());
    check(lib.router_topk_bwd(data(l), l.stride(0), static_cast<const int64_t*>(data(chosen)), data(dweights), dlogits.mutable_data_ptr(),
                              static_cast<int32_t>(l.size(0)), static_cast<int32_t>(l.size(1)), static_cast<int32_t>(chosen.size(1)), sigmoid,
                              renormalize, static_cast<float>(scale), dtype_code(l.scalar_type()), device, stream_of(device)),
          "b200moe_router_topk_bwd");
    return {dlogits};
  }
};

std::pair<Tensor, Tensor> router_topk(const Tensor& logits, int64_t top_k, const std::string& scoring, const std::optional<Tensor>& bias,
                                      int64_t num_groups, int64_t top_groups, bool renormalize, double scale) {
  TORCH_CHECK(logits.is_cuda(), "router_topk needs CUDA tensors (the sm_100a library is the only code path)");
  TORCH_CHECK_TYPE(dtype_code(logits.scalar_type()) >= 0, "router_topk supports bfloat16, float16 and float32 logits, got ", logits.dtype());
  TORCH_CHECK_VALUE(logits.dim() == 2, "router_topk: logits must be (tokens, experts), got ", logits.sizes());
  TORCH_CHECK_VALUE(scoring == "softmax" || scoring == "sigmoid", "router_topk: scoring must be 'softmax' or 'sigmoid', got '", scoring, "'");
  const int64_t experts = logits.size(1);
  TORCH_CHECK_VALUE(experts >= 1 && experts <= B200MOE_ROUTER_MAX_EXPERTS, "router_topk: 1 to ", B200MOE_ROUTER_MAX_EXPERTS, " experts, got ", experts);
  TORCH_CHECK_VALUE(num_groups >= 1 && num_groups <= B200MOE_ROUTER_MAX_GROUPS && experts % num_groups == 0 && top_groups >= 1 &&
                        top_groups <= num_groups,
                    "router_topk: ", experts, " experts cannot form ", num_groups, " equal groups of which ", top_groups, " are eligible");
  const int64_t eligible = experts / num_groups * top_groups;
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= std::min<int64_t>(B200MOE_ROUTER_MAX_TOP_K, eligible), "router_topk: cannot choose ", top_k, " of ",
                    eligible, " eligible experts (at most ", B200MOE_ROUTER_MAX_TOP_K, ")");
  TORCH_CHECK_VALUE(logits.size(0) <= std::numeric_limits<int32_t>::max(), "router_topk: ", logits.size(0), " tokens");
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == experts && bias->device() == logits.device() && bias->is_floating_point(),
                      "router_topk: bias must be ", experts, " floating point values on ", logits.device());
    // (the kernels read it as fp32, where every value of these types is itself)
    TORCH_CHECK_TYPE(dtype_code(bias->scalar_type()) >= 0, "router_topk: bias must be bfloat16, float16 or float32, got ", bias->dtype());
  }
  check_not_traced("router_topk");
  check_memory(logits, bias);
  check_no_tangent("router_topk", logits, bias);
  const Routing how{top_k, num_groups, top_groups, scoring == "sigmoid", renormalize, scale};
  const bool differentiable = at::GradMode::is_enabled() && logits.requires_grad();
  at::NoGradGuard no_grad;   // the choice has no gradient: nothing that leads to it is recorded
  const Tensor rows = row_major(logits);
  auto [weights, indices] = router_forward(rows, bias, how);
  if (differentiable) {
    auto node = new_node<RouterTopkBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->experts = experts;
    node->sigmoid = how.sigmoid;
    node->renormalize = renormalize;
    node->scale = scale;
    torch::autograd::set_history(weights, node);
    node->logits = SavedVariable(rows, false);
    node->indices = SavedVariable(indices, false);
  }
  return {weights, indices};
}

// ---------------------------------------------------------------- clip

// The bytes that a strided tensor takes: `size` of them at every sum of multiples of the dimensions' strides.
struct Span {
  struct Dim {
    int64_t stride, n;
  };
  int64_t begin = 0, bytes = 0, size = 0;   // from the first byte to behind the last one; of an element
  std::vector<Dim> dims;                    // of more than one index, the largest stride first
  explicit Span(const Tensor& t) {
    size = static_cast<int64_t>(t.element_size());
    if (t.numel() == 0) return;
    begin = reinterpret_cast<int64_t>(t.const_data_ptr());
    bytes = size;
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1 && t.stride(d) > 0) {   // (a stride of 0 adds no byte)
        dims.push_back({t.stride(d) * size, t.size(d)});
        bytes += dims.back().stride * (dims.back().n - 1);
      }
    std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
  }
};

// Whether no byte of `a` is one of `b`, which lies `shift` behind it: the indices of the largest stride S differ by k, and for each k
// that brings the rest of the two near each other, that rest is compared, k * S further on.  Where strides nest, as in
// slices and permutations of one buffer, that is a few steps; where `steps` run out the answer is no.
bool apart(const Span::Dim* a, const Span::Dim* a_end, int64_t a_bytes, const Span::Dim* b, const Span::Dim* b_end, int64_t b_bytes, int64_t shift,
           int& steps) {
  if (shift >= a_bytes || shift + b_bytes <= 0) return true;
  if ((a == a_end && b == b_end) || --steps < 0) return false;
  const int64_t s = std::max(a != a_end ? a->stride : 0, b != b_end ? b->stride : 0);
  int64_t least = 0, most = 0;   // k: b's index less a's
  if (a != a_end && a->stride == s) {
    least = -(a->n - 1);
    a_bytes -= (a++->n - 1) * s;
  }
  if (b != b_end && b->stride == s) {
    most = b->n - 1;
    b_bytes -= (b++->n - 1) * s;
  }
  const auto down = [s](int64_t v) { return v >= 0 ? v / s : -((-v + s - 1) / s); };
  least = std::max(least, down(-b_bytes - shift) + 1);
  most = std::min(most, down(a_bytes - 1 - shift));
  for (int64_t k = least; k <= most; ++k)
    if (!apart(a, a_end, a_bytes, b, b_end, b_bytes, shift + k * s, steps)) return false;
  return true;
}
constexpr int kApartSteps = 1 << 14;

bool share_memory(const Span& a, const Span& b) {
  int steps = kApartSteps;
  return a.bytes != 0 && b.bytes != 0 &&
         !apart(a.dims.data(), a.dims.data() + a.dims.size(), a.bytes, b.dims.data(), b.dims.data() + b.dims.size(), b.bytes, b.begin - a.begin, steps);
}
// Whether two elements of a tensor share memory (but for strides of 0).
bool shares_with_itself(const Span& t) {
  int64_t rest = t.bytes;
  const Span::Dim* end = t.dims.data() + t.dims.size();
  for (const Span::Dim* d = t.dims.data(); d != end; ++d) {
    rest -= (d->n - 1) * d->stride;
    for (int64_t k = 1; k < d->n && k * d->stride < rest; ++k) {
      int steps = kApartSteps;
      if (!apart(d + 1, end, rest, d + 1, end, rest, k * d->stride, steps)) return true;
    }
  }
  return false;
}

// Whether the library gets a tensor itself; otherwise a copy, which dense() makes.
bool goes_itself(const Tensor& t) { return t.is_contiguous() && !t.is_neg(); }
Tensor dense(const Tensor& t) { return goes_itself(t) ? t : as_it_lies(t).contiguous(); }

// Refuses tensors to be written that have memory twice, share it with one another or with one that is read.  What goes to the library
// itself is looked through there.
void check_apart(const char* name, const std::vector<Tensor>& written, const std::vector<Tensor>& read) {
  for (const Tensor& t : written) {
    if (goes_itself(t)) continue;
    for (int64_t d = 0; d < t.dim(); ++d)
      TORCH_CHECK_VALUE(t.stride(d) != 0 || t.size(d) <= 1, name, ": a tensor with a stride of 0 cannot be written in place");
    TORCH_CHECK_VALUE(!shares_with_itself(Span(t)), name, ": a tensor whose elements share memory cannot be written in place");
  }
  std::vector<std::pair<Span, bool>> all;   // and whether it is written
  int64_t low = std::numeric_limits<int64_t>::max(), high = 0;
  const auto copied = [&](const std::vector<Tensor>& tensors, bool writes) {
    for (const Tensor& t : tensors) {
      if (goes_itself(t)) continue;
      all.emplace_back(Span(t), writes);
      if (t.numel() == 0) continue;
      low = std::min(low, all.back().first.begin);
      high = std::max(high, all.back().first.begin + all.back().first.bytes);
    }
  };
  copied(written, true);
  copied(read, false);
  const auto near = [&](const std::vector<Tensor>& tensors, bool writes) {   // and the others that one of those could reach
    for (const Tensor& t : tensors) {
      const int64_t begin = reinterpret_cast<int64_t>(t.const_data_ptr());
      if (goes_itself(t) && begin < high && begin + t.numel() * static_cast<int64_t>(t.element_size()) > low) all.emplace_back(Span(t), writes);
    }
  };
  near(written, true);
  near(read, false);
  std::sort(all.begin(), all.end(), [](const auto& a, const auto& b) { return a.first.begin < b.first.begin; });
  for (size_t i = 0; i < all.size(); ++i)
    for (size_t j = i + 1; j < all.size() && all[j].first.begin < all[i].first.begin + all[i].first.bytes; ++j)
      if (all[i].second || all[j].second) {
        const int rc = share_memory(all[i].first, all[j].first) ? B200TRAIN_EOVERLAP : 0;
        check(rc, name);
      }
}

// The arrays that the library reads: addresses, counts and types of contiguous tensors on one device.
struct Table {
  std::vector<int64_t> grads, params, counts;
  std::vector<int32_t> dtypes;
  int device = -1;
  Table(const char* name, const std::vector<Tensor>& g, const std::vector<Tensor>* p) {
    const size_t n = g.size();
    grads.resize(n);
    counts.resize(n);
    dtypes.resize(n);
    if (p != nullptr) params.resize(n);
    device = g[0].is_cuda() ? static_cast<int>(g[0].get_device()) : -1;
    for (size_t i = 0; i < n; ++i) {
      TORCH_CHECK(device >= 0 && g[i].is_cuda() && g[i].get_device() == device && (p == nullptr || ((*p)[i].is_cuda() && (*p)[i].get_device() == device)),
                  name, " needs CUDA tensors on one device (the sm_100a library is the only code path)");
      TORCH_CHECK_TYPE(g[i].layout() == at::kStrided, name, " supports strided tensors, got ", g[i].layout());
      dtypes[i] = dtype_code(g[i].scalar_type());
      TORCH_CHECK_TYPE(dtypes[i] >= 0, name, " supports bfloat16, float16 and float32, got ", g[i].dtype());
      counts[i] = g[i].numel();
      grads[i] = reinterpret_cast<int64_t>(address(g[i]));
      if (p != nullptr) params[i] = reinterpret_cast<int64_t>(address((*p)[i]));
    }
  }
};

struct Output {
  Tensor scratch, norm;
  int64_t doubles;
  Output(const Tensor& like, size_t tensors, int device) {
    doubles = lib.clip_scratch_doubles(static_cast<int64_t>(tensors), device);
    scratch = empty_on(like, {doubles}, at::kDouble);
    norm = empty_on(like, {}, at::kFloat);
  }
};

float limit_of(const char* name, double max_norm) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, name, ": max_norm must not be negative, got ", max_norm);
  return static_cast<float>(max_norm);
}

Tensor global_grad_norm(const std::vector<Tensor>& tensors) {
  at::NoGradGuard no_grad;
  check_not_traced("global_grad_norm");
  if (tensors.empty()) return at::zeros({}, at::kFloat);
  std::vector<Tensor> packed;
  packed.reserve(tensors.size());
  const bool tangents = tangents_exist();
  for (const Tensor& t : tensors) {
    if (tangents) check_no_tangent("global_grad_norm", t);
    packed.push_back(dense(t));
  }
  const Table t("global_grad_norm", packed, nullptr);
  Output out(packed[0], packed.size(), t.device);
  check(lib.grad_norm(t.grads.data(), t.counts.data(), t.dtypes.data(), static_cast<int64_t>(packed.size()), out.scratch.mutable_data_ptr<double>(),
                      out.doubles, out.norm.mutable_data_ptr<float>(), t.device, stream_of(t.device)),
        "b200train_grad_norm");
  return out.norm;
}

Tensor clip_grad_norm(const std::vector<Tensor>& parameters, double max_norm) {
  at::NoGradGuard no_grad;
  check_not_traced("clip_grad_norm");
  const float limit = limit_of("clip_grad_norm", max_norm);
  std::vector<Tensor> grads, packed;
  const bool tangents = tangents_exist();
  bool copied = false;
  grads.reserve(parameters.size());
  packed.reserve(parameters.size());
  for (const Tensor& p : parameters) {
    const Tensor& g = p.grad();
    if (!g.defined()) continue;
    if (tangents) check_no_tangent("clip_grad_norm", g);
    grads.push_back(g);
    packed.push_back(g.layout() == at::kStrided ? dense(g) : g);
    copied = copied || !packed.back().is_same(g);
  }
  if (grads.empty()) return at::zeros({}, at::kFloat);
  const Table t("clip_grad_norm", packed, nullptr);
  if (copied) check_apart("clip_grad_norm", grads, {});
  Output out(packed[0], packed.size(), t.device);
  check(lib.clip_grads(t.grads.data(), t.counts.data(), t.dtypes.data(), static_cast<int64_t>(packed.size()), limit,
                       out.scratch.mutable_data_ptr<double>(), out.doubles, out.norm.mutable_data_ptr<float>(), t.device, stream_of(t.device)),
        "b200train_clip_grads");
  for (size_t i = 0; i < grads.size(); ++i) {
    if (packed[i].is_same(grads[i])) grads[i].unsafeGetTensorImpl()->bump_version();
    else grads[i].copy_(packed[i]);
  }
  return out.norm;
}

Tensor clipped_sgd_step(const std::vector<Tensor>& parameters, double lr, double max_norm) {
  at::NoGradGuard no_grad;
  check_not_traced("clipped_sgd_step");
  const float limit = limit_of("clipped_sgd_step", max_norm);
  std::vector<Tensor> params, grads, packed;
  const bool tangents = tangents_exist();
  bool copied = false;
  for (const Tensor& p : parameters) {
    const Tensor& g = p.grad();
    if (!g.defined()) continue;
    if (tangents) check_no_tangent("clipped_sgd_step", p, g);
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), "clipped_sgd_step: a gradient must have its parameter's type, got ", g.dtype(), " for ",
                     p.dtype());
    params.push_back(p);
    grads.push_back(g.layout() == at::kStrided ? dense(g) : g);
    packed.push_back(dense(p));
    copied = copied || !grads.back().is_same(g) || !packed.back().is_same(p);
  }
  if (params.empty()) return at::zeros({}, at::kFloat);
  const Table t("clipped_sgd_step", grads, &packed);
  if (copied) {
    std::vector<Tensor> read;
    for (const Tensor& p : params) read.push_back(p.grad());
    check_apart("clipped_sgd_step", params, read);
  }
  Output out(grads[0], grads.size(), t.device);
  check(lib.clipped_sgd(t.grads.data(), t.params.data(), t.counts.data(), t.dtypes.data(), static_cast<int64_t>(grads.size()),
                        static_cast<float>(lr), limit, out.scratch.mutable_data_ptr<double>(), out.doubles, out.norm.mutable_data_ptr<float>(),
                        t.device, stream_of(t.device)),
        "b200train_clipped_sgd");
  for (size_t i = 0; i < params.size(); ++i) {
    if (packed[i].is_same(params[i])) params[i].unsafeGetTensorImpl()->bump_version();
    else params[i].copy_(packed[i]);
  }
  return out.norm;
}

}  // namespace

PYBIND11_MODULE(_train_binding, m) {
  m.def("set_library", &set_library);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("rms_norm", &rms_norm);
  m.def("router_topk", &router_topk);
  m.def("global_grad_norm", &global_grad_norm);
  m.def("clip_grad_norm", &clip_grad_norm);
  m.def("clipped_sgd_step", &clipped_sgd_step);
  m.def("share_memory", [](const Tensor& a, const Tensor& b) { return share_memory(Span(a), Span(b)); });
  m.def("shares_with_itself", [](const Tensor& t) { return shares_with_itself(Span(t)); });
}
