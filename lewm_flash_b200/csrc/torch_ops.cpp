// The training operators as torch functions: argument checks, strides, allocation, streams and
// autograd around the C ABI of lewm_b200.h (lewm_norm_*, lewm_grad_*), as the Python extension
// module lewm_flash_b200._torch_ops. lewm_flash_b200/training.py is the documented surface.
//
// In C++ because a training step calls these operators a hundred times on rows that take the GPU
// a few microseconds. Host time of a forward and backward pass (900 x 192 float32): through a
// Python autograd.Function and ctypes 140 us, through this module's autograd node 62 us (45 of
// them the autograd engine's own); a forward pass alone 15 and 4 us; a clip of 523 tensors, with
// its checks, 677 and 48 us.
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <numeric>
#include <optional>
#include <vector>

#include "lewm_b200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

// ------------------------------------------------------------------ checks
int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return LEWM_TYPE_F32;
    case at::kBFloat16: return LEWM_TYPE_BF16;
    case at::kHalf: return LEWM_TYPE_F16;
    default: return -1;
  }
}

// A tracer (torch.jit.trace, make_fx, torch.export) records what goes through torch's dispatcher. It
// does not see these calls and would take their outputs for constants.
void check_no_tracer() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  const bool tracing = at::tracer::impl::is_dispatch_enabled() ||
                       c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                       TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value() ||
                       TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL).has_value() ||
                       TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE).has_value();
  TORCH_CHECK_NOT_IMPLEMENTED(!tracing, "the B200 training operators cannot be traced: trace the model without them "
                              "(install_training_norms(...).remove())");
}

// Whether tensors can have tangents at all: a level of torch.autograd.forward_ad is open. Asked once per
// call; a look at each of 1046 tensors took a clip of 523 from 52 to 115 us.
bool forward_mode() {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
         torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
}

// A tangent, which the kernels would drop.
bool has_tangent(const Tensor& t) { return forward_mode() && t._fw_grad(0).defined(); }

void check_no_tangent(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), name, " has a tangent: the B200 training operators have no "
                              "forward-mode derivative");
}

// Tensors that stand for others, with no memory of their own or not theirs alone to interpret: what
// torch.func's transforms (vmap, grad, functionalize) and batched gradients pass in, and subclasses with a
// __torch_dispatch__ (DTensor, FakeTensor).
bool is_wrapper(const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet keys({DispatchKey::FuncTorchBatched, DispatchKey::BatchedNestedTensor,
                                      DispatchKey::Batched, DispatchKey::FuncTorchGradWrapper,
                                      DispatchKey::Functionalize, DispatchKey::Python, DispatchKey::ZeroTensor});
  return t.key_set().has_any(keys);
}

void check_no_wrapper(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!is_wrapper(t), name, " belongs to a transform (torch.func, vmap, batched gradients) or "
                              "is a subclass with a __torch_dispatch__: the B200 training operators take plain tensors");
}

void check_tensor(const char* name, const Tensor& t) {
  check_no_wrapper(name, t);
  TORCH_CHECK_VALUE(type_code(t) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " must be a dense tensor, got layout ", t.layout());
  TORCH_CHECK_VALUE(!t.is_neg(), name, " is a lazily negated view: pass it through resolve_neg()");
  check_no_tangent(name, t);
}

void check_same_device(const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", x on ", x.device());
}

void need_cuda(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "the B200 training operators need a CUDA device, got ", t.device());
}

float check_eps(double eps) {
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < std::numeric_limits<double>::infinity(), "eps must be finite and >= 0, got ",
                    eps);
  return static_cast<float>(eps);
}

// Raises the package's LewmError for a failed C-ABI call made with the GIL held; in a backward pass
// (an engine thread) the error becomes a RuntimeError with the same text.
void check_status(lewm_status s, bool in_backward = false) {
  if (s == LEWM_OK) return;
  const char* msg = lewm_last_error(nullptr);
  TORCH_CHECK(!in_backward, "lewm_b200 status ", static_cast<int>(s), ": ", msg);
  py::object lib = py::module_::import("lewm_flash_b200._lib");
  py::object type = lib.attr(s == LEWM_INVALID_ARG ? "LewmInvalidArgument" : "LewmError");
  PyErr_SetObject(type.ptr(), type(static_cast<int>(s), msg).ptr());
  throw py::error_already_set();
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// A contiguous tensor on the device of `like`, past the dispatcher: a forward pass
// with two of them takes 6.4 us of host time, with at::empty 7.0.
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// ------------------------------------------------------------------ rows
struct Rows {
  Tensor t;
  int64_t stride;
};

// `t` as rows of its last dim and the elements between them, copied only where the leading dims do
// not step evenly through memory or the last dim is not dense.
Rows rows_of(const Tensor& t) {
  const auto size = t.sizes(), stride = t.strides();
  const int64_t last = t.dim() - 1;
  if (t.is_contiguous()) return {t, size[last]};
  if (stride[last] == 1 || size[last] == 1) {
    int64_t step = -1, extent = 1;  // stride of the rows so far, and how many there are
    bool even = true;
    for (int64_t d = last - 1; d >= 0 && even; --d) {
      if (size[d] == 1) continue;
      if (step < 0) step = stride[d];
      else even = stride[d] == step * extent;
      extent *= size[d];
    }
    if (even) return {t, step < 0 ? size[last] : step};
  }
  return {t.contiguous(), size[last]};
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// ------------------------------------------------------------------ norms
// y = z a + b (group 0) or z (1 + a) + b with a row of a and b for `group` rows of x. x is `rows_of`.
Tensor norm_forward(const Rows& x, const Tensor& a, const Tensor& b, float eps, int64_t group, float* stats) {
  const int64_t width = x.t.size(-1), rows = x.t.numel() / width;
  Tensor y = empty(x.t.sizes(), x.t.scalar_type(), x.t);
  if (rows == 0) return y;
  const Rows ra = a.defined() ? rows_of(a) : Rows{}, rb = b.defined() ? rows_of(b) : Rows{};
  const int p_type = a.defined() ? type_code(a) : b.defined() ? type_code(b) : LEWM_TYPE_F32;
  const lewm_norm_desc d{rows, width, x.stride, group, ra.stride, rb.stride, type_code(x.t), p_type, eps};
  check_status(lewm_norm_forward(&d, x.t.const_data_ptr(), ptr(ra.t), ptr(rb.t), y.mutable_data_ptr(), stats,
                                 x.t.get_device(), stream_of(x.t)));
  return y;
}

struct NormBackward : public torch::autograd::Node {
  SavedVariable x_, a_;
  Tensor stats_;
  float eps = 0.f;
  int64_t group = 0;
  std::vector<int64_t> x_shape, a_shape, b_shape;
  at::ScalarType p_type = at::kFloat;
  bool has_a = false, has_b = false;

  std::string name() const override { return "LewmNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x_.reset_data();
    a_.reset_data();
    stats_.reset();
  }

  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    Tensor dy = std::move(grads[0]);
    const bool need_x = task_should_compute_output(0), need_a = has_a && task_should_compute_output(1),
               need_b = has_b && task_should_compute_output(2);
    if (!dy.defined() || !(need_x || need_a || need_b)) return out;
    check_no_tracer();
    check_no_wrapper("the output's gradient", dy);
    check_no_tangent("the output's gradient", dy);
    Tensor x, a, stats;
    {
      std::lock_guard<std::mutex> lock(mutex_);
      x = x_.unpack();
      if (has_a) a = a_.unpack();
      stats = stats_;
    }
    const bool twice = at::GradMode::is_enabled();  // create_graph: a second pass would need our derivative
    {
      at::NoGradGuard no_grad;
      if (dy.is_neg()) dy = dy.resolve_neg();
      const int64_t width = x_shape.back(), rows = x.numel() / width;
      if (need_x) out[0] = empty(x_shape, x.scalar_type(), x);
      // A shift row per row of x: its gradient is dy, and may be dy's memory if nobody else holds that
      // (the caller, another branch of the graph, a hook); else the kernel writes a copy.
      const bool dy_is_db = need_b && group == 1 && rows > 0 && p_type == dy.scalar_type() && !twice &&
                            dy.is_contiguous() && dy.use_count() == 1 && dy.has_storage() && dy.storage().use_count() == 1;
      if (rows == 0) {
        if (need_a) out[1] = empty(a_shape, p_type, x).zero_();
        if (need_b) out[2] = empty(b_shape, p_type, x).zero_();
      } else {
        if (need_a) out[1] = empty(a_shape, p_type, x);
        if (need_b && !dy_is_db) out[2] = empty(b_shape, p_type, x);
        if (need_x || need_a || out[2].defined()) {
          const Rows rx = rows_of(x), rd = rows_of(dy), ra = a.defined() ? rows_of(a) : Rows{};
          const int p = p_type == at::kFloat ? LEWM_TYPE_F32 : p_type == at::kBFloat16 ? LEWM_TYPE_BF16 : LEWM_TYPE_F16;
          const lewm_norm_desc d{rows, width, rx.stride, group, ra.stride, 0, type_code(x), p, eps};
          const size_t bytes = need_a || out[2].defined() ? lewm_norm_workspace(&d) : 0;
          Tensor ws;
          if (bytes) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, x);
          check_status(lewm_norm_backward(&d, rd.t.const_data_ptr(), rd.stride, rx.t.const_data_ptr(), ptr(ra.t),
                                          static_cast<const float*>(stats.const_data_ptr()), mut(out[0]), mut(out[1]),
                                          mut(out[2]), mut(ws), bytes, x.get_device(), stream_of(x)),
                       true);
        }
        if (dy_is_db) out[2] = dy.sizes() == at::IntArrayRef(b_shape) ? std::move(dy) : dy.view(b_shape);
      }
    }
    if (twice) {
      variable_list defined;
      for (auto& t : out)
        if (t.defined()) defined.push_back(t.detach().requires_grad_(true));
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "the B200 norms are differentiable once: their gradients cannot be differentiated", defined.size());
      defined = (*error)(std::move(defined));
      size_t i = 0;
      for (auto& t : out)
        if (t.defined()) t = defined[i++];
    }
    return out;
  }
};

Tensor norm(const Tensor& x, const Tensor& a, const Tensor& b, float eps, int64_t group) {
  need_cuda(x);
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || (a.defined() && a.requires_grad()) ||
                                                   (b.defined() && b.requires_grad()));
  if (!grad) {
    at::NoGradGuard no_grad;
    return norm_forward(rows_of(x), a, b, eps, group, nullptr);
  }
  auto node = std::shared_ptr<NormBackward>(new NormBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, a, b));
  Tensor y;
  {
    at::NoGradGuard no_grad;
    const Rows rx = rows_of(x);  // a copy, where one is needed, serves the backward pass too
    const int64_t rows = x.numel() / x.size(-1);
    node->stats_ = empty({2, rows}, at::kFloat, x);
    y = norm_forward(rx, a, b, eps, group, static_cast<float*>(node->stats_.mutable_data_ptr()));
    node->x_ = SavedVariable(rx.t, false);
    if (a.defined()) node->a_ = SavedVariable(a, false);
  }
  node->eps = eps;
  node->group = group;
  node->x_shape = x.sizes().vec();
  node->has_a = a.defined();
  node->has_b = b.defined();
  if (a.defined()) node->a_shape = a.sizes().vec(), node->p_type = a.scalar_type();
  if (b.defined()) node->b_shape = b.sizes().vec(), node->p_type = b.scalar_type();
  torch::autograd::set_history(y, node);
  return y;
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  check_no_tracer();
  check_tensor("x", x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "x must have a last dim of at least 1, got shape ", x.sizes());
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  auto check_param = [&](const char* name, const Tensor& p) {
    if (!p.defined()) return;
    check_tensor(name, p);
    check_same_device(name, p, x);
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == x.size(-1), name, " must be (", x.size(-1), ",), got ", p.sizes());
  };
  check_param("weight", w);
  check_param("bias", b);
  if (w.defined() && b.defined())
    TORCH_CHECK_VALUE(w.scalar_type() == b.scalar_type(), "weight and bias must have one type, got ", w.scalar_type(),
                      " and ", b.scalar_type());
  return norm(x, w, b, check_eps(eps), 0);
}

Tensor ada_layer_norm(const Tensor& x, const Tensor& shift, const Tensor& scale, double eps) {
  check_no_tracer();
  check_tensor("x", x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "x must have a last dim of at least 1, got shape ", x.sizes());
  check_tensor("shift", shift);
  check_tensor("scale", scale);
  check_same_device("shift", shift, x);
  check_same_device("scale", scale, x);
  TORCH_CHECK_VALUE(shift.sizes() == scale.sizes() && shift.scalar_type() == scale.scalar_type(),
                    "shift and scale must have one shape and type, got ", shift.sizes(), " ", shift.scalar_type(),
                    " and ", scale.sizes(), " ", scale.scalar_type());
  int64_t group = 1;
  if (shift.sizes() != x.sizes()) {
    const int64_t n = x.dim(), pad = n - shift.dim();
    auto m = [&](int64_t d) { return d < pad ? int64_t{1} : shift.size(d - pad); };
    bool fits = pad >= 0 && shift.dim() > 0 && shift.size(-1) == x.size(-1);
    int64_t d = n - 2;
    for (; fits && d >= 0 && m(d) == 1; --d) group *= x.size(d);
    for (; fits && d >= 0; --d) fits = m(d) == x.size(d);
    TORCH_CHECK_VALUE(fits, "shift and scale of shape ", shift.sizes(), " do not modulate x of shape ", x.sizes(),
                      ": give a row per row of x, or size 1 in the dims before the last");
  }
  if (x.numel() == 0) group = 1;  // no rows
  return norm(x, scale, shift, check_eps(eps), group);
}

// ------------------------------------------------------------------ gradient norm and clipping
int norm_kind(double norm_type) {
  if (norm_type == 2.0) return LEWM_NORM_L2;
  TORCH_CHECK_VALUE(norm_type == std::numeric_limits<double>::infinity(), "norm_type must be 2 or inf, got ",
                    norm_type);
  return LEWM_NORM_MAX;
}

float check_max_norm(double max_norm) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must be >= 0, got ", max_norm);
  return static_cast<float>(max_norm);
}

// The tensors of a Python list, borrowed from it: converting a list through the binding's casters
// took longer than all the checks.
using Refs = std::vector<const Tensor*>;
Refs refs(const char* name, const py::list& list) {
  Refs out;
  out.reserve(list.size());
  for (py::handle h : list) {
    TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), name, "[", out.size(), "] must be a tensor, got ",
                     Py_TYPE(h.ptr())->tp_name);
    out.push_back(&THPVariable_Unpack(h.ptr()));
  }
  return out;
}

void check_list(const char* name, const Refs& ts) {
  const bool tangents = forward_mode();
  for (size_t i = 0; i < ts.size(); ++i) {
    const Tensor& t = *ts[i];
    if (type_code(t) < 0 || t.layout() != at::kStrided || t.is_neg() || is_wrapper(t) || (tangents && has_tangent(t)))
      check_tensor((std::string(name) + "[" + std::to_string(i) + "]").c_str(), t);
    TORCH_CHECK_VALUE(t.device() == ts[0]->device(), name, "[", i, "] is on ", t.device(), ", ", name, "[0] on ",
                      ts[0]->device(), ": one device per call");
  }
}

// Whether any destination [dst, dst + size) meets another destination or another tensor's source.
bool overlap(const std::vector<int64_t>& src, const std::vector<int64_t>& dst, const std::vector<int64_t>& size) {
  std::vector<std::pair<int64_t, int64_t>> out;
  out.reserve(dst.size());
  for (size_t i = 0; i < dst.size(); ++i)
    if (size[i] > 0) out.emplace_back(dst[i], dst[i] + size[i]);
  std::sort(out.begin(), out.end());
  for (size_t i = 1; i < out.size(); ++i)
    if (out[i - 1].second > out[i].first) return true;
  // Destinations are disjoint and sorted: those a source meets are a run of them; only its own
  // destination, lying exactly on it, may be in there.
  for (size_t i = 0; i < src.size(); ++i) {
    if (size[i] <= 0) continue;
    auto first = std::upper_bound(out.begin(), out.end(), src[i],
                                  [](int64_t v, const std::pair<int64_t, int64_t>& o) { return v < o.second; });
    auto last = std::lower_bound(first, out.end(), src[i] + size[i],
                                 [](const std::pair<int64_t, int64_t>& o, int64_t v) { return o.first < v; });
    if (last - first != (src[i] == dst[i] ? 1 : 0)) return true;
  }
  return false;
}

// The bytes of a strided tensor: runs of `run` bytes from `base` on, at all sums of multiples of the
// strides, the largest first. Each stride reaches past all that lies under it, so no two elements meet.
struct Region {
  struct Dim {
    int64_t stride, size, inner;  // bytes; inner: from first to last byte of what lies under the dim
  };
  int64_t base = 0, run = 0, span = 0;
  std::vector<Dim> dims;
  bool own_overlap = false;

  explicit Region(const Tensor& t) : base(reinterpret_cast<int64_t>(t.const_data_ptr())) {
    if (t.numel() == 0) return;
    std::vector<std::pair<int64_t, int64_t>> by_stride;
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1) by_stride.emplace_back(t.stride(d) * t.element_size(), t.size(d));
    std::sort(by_stride.begin(), by_stride.end());
    run = span = t.element_size();
    for (const auto& [stride, size] : by_stride) {
      own_overlap |= stride < span;
      if (dims.empty() && stride == run) run = span = run * size;
      else dims.push_back({stride, size, span}), span += (size - 1) * stride;
    }
    std::reverse(dims.begin(), dims.end());
  }
};

// Whether the parts of a and b from their dims i and j on, at x and y, share a byte. Gives up with true
// after `steps` splits.
bool meet(const Region& a, size_t i, int64_t x, const Region& b, size_t j, int64_t y, int64_t* steps) {
  const bool split_a = i < a.dims.size(), split_b = j < b.dims.size();
  const int64_t span_a = split_a ? a.dims[i].inner + (a.dims[i].size - 1) * a.dims[i].stride : a.run;
  const int64_t span_b = split_b ? b.dims[j].inner + (b.dims[j].size - 1) * b.dims[j].stride : b.run;
  if (x >= y + span_b || y >= x + span_a) return false;
  if (!split_a && !split_b) return true;
  if (--*steps < 0) return true;
  // Runs that are apart modulo a divisor of all strides are apart: columns of one buffer.
  int64_t g = 0;
  for (size_t k = i; k < a.dims.size(); ++k) g = std::gcd(g, a.dims[k].stride);
  for (size_t k = j; k < b.dims.size(); ++k) g = std::gcd(g, b.dims[k].stride);
  const int64_t from = ((y - x) % g + g) % g;  // of b's run behind a's, round the circle
  if (from >= a.run && from + b.run <= g) return false;
  // Split the one that spans more; only its parts near the other one.
  if (!split_a || (split_b && span_b > span_a)) return meet(b, j, y, a, i, x, steps);
  const Region::Dim& d = a.dims[i];
  const int64_t after = y - x - d.inner;  // a part that starts at or before it ends before b begins
  const int64_t first = after < 0 ? 0 : after / d.stride + 1, last = std::min(d.size - 1, (y + span_b - 1 - x) / d.stride);
  for (int64_t k = first; k <= last; ++k)
    if (meet(a, i + 1, x + k * d.stride, b, j, y, steps)) return true;
  return false;
}

// Refuses gradients, some of them strided, that share memory with each other or within themselves.
void check_apart(const Refs& grads) {
  std::vector<Region> regions;
  regions.reserve(grads.size());
  for (const Tensor* g : grads) {
    if (g->numel() == 0) continue;
    regions.emplace_back(*g);
    TORCH_CHECK_VALUE(!regions.back().own_overlap, "a gradient of shape ", g->sizes(), " and strides ", g->strides(),
                      " shares memory between its own elements");
  }
  std::sort(regions.begin(), regions.end(), [](const Region& a, const Region& b) { return a.base < b.base; });
  int64_t steps = int64_t{1} << 22;
  for (size_t i = 0; i < regions.size(); ++i)
    for (size_t j = i + 1; j < regions.size() && regions[j].base < regions[i].base + regions[i].span; ++j)
      TORCH_CHECK_VALUE(!meet(regions[i], 0, regions[i].base, regions[j], 0, regions[j].base, &steps),
                        "gradients overlap in memory (the same one listed twice?), or are too finely interleaved "
                        "to tell");
}

// The kernels' call: norm of dense `src`, and with `dst` their scaled copies.
Tensor clip(const Refs& src, const Refs* dst, float max_norm, int kind, const Tensor& norm_in) {
  const size_t n = src.size();
  std::vector<const void*> sp(n);
  std::vector<void*> dp(dst ? n : 0);
  std::vector<int64_t> count(n);
  std::vector<int32_t> type(n);
  for (size_t i = 0; i < n; ++i) {
    count[i] = src[i]->numel();
    type[i] = type_code(*src[i]);
    sp[i] = src[i]->const_data_ptr();
    if (dst) dp[i] = (*dst)[i]->mutable_data_ptr();
  }
  if (dst) {
    std::vector<int64_t> s(n), d(n), size(n);
    for (size_t i = 0; i < n; ++i) {
      s[i] = reinterpret_cast<int64_t>(sp[i]);
      d[i] = reinterpret_cast<int64_t>(dp[i]);
      size[i] = count[i] * (type[i] == LEWM_TYPE_F32 ? 4 : 2);
    }
    TORCH_CHECK_VALUE(!overlap(s, d, size),
                      "gradients overlap in memory (the same one listed twice?), or an output overlaps one");
  }
  need_cuda(*src[0]);
  Tensor norm = empty({}, at::kFloat, *src[0]), ws = empty({LEWM_GRAD_WORKSPACE}, at::kByte, *src[0]);
  const int device = src[0]->get_device();
  void* stream = stream_of(*src[0]);
  float* out = static_cast<float*>(norm.mutable_data_ptr());
  const int32_t m = static_cast<int32_t>(std::min<size_t>(n, std::numeric_limits<int32_t>::max()));
  if (!dst) check_status(lewm_grad_norm(sp.data(), count.data(), type.data(), m, kind, mut(ws), out, device, stream));
  else
    check_status(lewm_grad_clip(sp.data(), dp.data(), count.data(), type.data(), m, kind, max_norm,
                                static_cast<const float*>(ptr(norm_in)), mut(ws), out, device, stream));
  return norm;
}

// `ts` with contiguous copies, held in `copies`, in the place of those that are not.
Refs dense(const Refs& ts, std::vector<Tensor>* copies) {
  Refs out = ts;
  copies->reserve(ts.size());  // the addresses of its elements stay
  for (size_t i = 0; i < ts.size(); ++i) {
    if (ts[i]->is_contiguous()) continue;
    copies->push_back(ts[i]->contiguous());
    out[i] = &copies->back();
  }
  return out;
}

// A change in place that autograd has to see.
void bump(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor grad_norm(const py::list& list, double norm_type) {
  check_no_tracer();
  at::NoGradGuard no_grad;
  const int kind = norm_kind(norm_type);
  const Refs grads = refs("grads", list);
  if (grads.empty()) return at::zeros({}, at::kFloat);
  check_list("grads", grads);
  std::vector<Tensor> copies;
  return clip(dense(grads, &copies), nullptr, 0.f, kind, Tensor());
}

std::pair<py::list, Tensor> clip_grads(const py::list& list, double max_norm, double norm_type,
                                       const std::optional<py::list>& out_given) {
  check_no_tracer();
  at::NoGradGuard no_grad;
  const int kind = norm_kind(norm_type);
  const float limit = check_max_norm(max_norm);
  const Refs grads = refs("grads", list);
  py::list out_list = out_given ? *out_given : py::list();
  if (out_given)
    TORCH_CHECK_VALUE(out_list.size() == grads.size(), "out has ", out_list.size(), " tensors, grads ", grads.size());
  if (grads.empty()) return {out_list, at::zeros({}, at::kFloat)};
  check_list("grads", grads);
  if (!out_given) {
    need_cuda(*grads[0]);
    for (const Tensor* g : grads) out_list.append(empty(g->sizes(), g->scalar_type(), *g));
  }
  const Refs out = refs("out", out_list);
  const bool tangents = forward_mode();
  for (size_t i = 0; out_given && i < grads.size(); ++i) {
    const Tensor &g = *grads[i], &o = *out[i];
    TORCH_CHECK_VALUE(o.layout() == at::kStrided && !o.is_neg() && o.sizes() == g.sizes() && o.scalar_type() == g.scalar_type() &&
                          o.device() == g.device(),
                      "out[", i, "] must be a ", g.scalar_type(), " tensor of shape ", g.sizes(), " on ", g.device());
    TORCH_CHECK_VALUE(o.is_contiguous(), "out[", i, "] must be contiguous");
    if (is_wrapper(o) || (tangents && has_tangent(o))) check_tensor(("out[" + std::to_string(i) + "]").c_str(), o);
  }
  std::vector<Tensor> copies;
  Tensor norm = clip(dense(grads, &copies), &out, limit, kind, Tensor());
  if (out_given)
    for (const Tensor* o : out) bump(*o);
  return {std::move(out_list), std::move(norm)};
}

Tensor clip_in_place(const py::list& list, double max_norm, double norm_type, bool error_if_nonfinite) {
  check_no_tracer();
  at::NoGradGuard no_grad;
  const int kind = norm_kind(norm_type);
  const float limit = check_max_norm(max_norm);
  const Refs grads = refs("grad", list);
  if (grads.empty()) return at::zeros({}, at::kFloat);
  check_list("grad", grads);
  Refs strided;
  for (const Tensor* g : grads)
    if (!g->is_contiguous()) strided.push_back(g);
  if (!strided.empty()) check_apart(grads);
  std::vector<Tensor> copies;
  const Refs ts = dense(grads, &copies);
  Tensor norm_in;
  if (error_if_nonfinite) {
    norm_in = clip(ts, nullptr, 0.f, kind, Tensor());
    TORCH_CHECK(std::isfinite(norm_in.item<float>()), "The total norm of order ", norm_type,
                " for gradients is non-finite, so it cannot be clipped");
  }
  Tensor norm = clip(ts, &ts, limit, kind, norm_in);
  for (size_t i = 0; i < strided.size(); ++i) strided[i]->copy_(copies[i]);  // counts as a change by itself
  for (const Tensor* g : grads)
    if (g->is_contiguous()) bump(*g);
  return norm;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.attr("abi_version") = LEWM_ABI_VERSION;
  m.def("layer_norm", torch::wrap_pybind_function(layer_norm), py::arg("x"), py::arg("weight"), py::arg("bias"),
        py::arg("eps"));
  m.def("ada_layer_norm", torch::wrap_pybind_function(ada_layer_norm), py::arg("x"), py::arg("shift"),
        py::arg("scale"), py::arg("eps"));
  m.def("grad_norm", torch::wrap_pybind_function(grad_norm), py::arg("grads"), py::arg("norm_type"));
  m.def("clip_grads", torch::wrap_pybind_function(clip_grads), py::arg("grads"), py::arg("max_norm"),
        py::arg("norm_type"), py::arg("out"));
  m.def("clip_in_place", torch::wrap_pybind_function(clip_in_place), py::arg("grads"), py::arg("max_norm"),
        py::arg("norm_type"), py::arg("error_if_nonfinite"));
  // For tests: how a tensor's rows are read, and the overlap rule.
  m.def("rows", [](const Tensor& t) {
    Rows r = rows_of(t);
    return std::make_pair(r.t, r.stride);
  });
  m.def("overlap", overlap);
}
