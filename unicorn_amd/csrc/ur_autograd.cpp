// ur_autograd.cpp -- autograd nodes of the operators of the networks around the renderer, over the C ABI of
// include/unicorn_render.h.
//
// The renderer's own nodes are Python (unicorn_amd/ops.py): one pair of calls per step of 0.1 ms and more.  These operators are
// called many times a step on small tensors, where the host is what counts: the autograd engine runs a backward on a thread of
// its own, and Python code there costs twice what it costs on the caller's thread (measured: 192 x 512, forward and
// backward, 118 us with Python nodes, of which 60 us in Python).  Shapes, types and devices are checked by the Python layer;
// here tensors are allocated, laid out as rows and handed over as pointers.  The library is the one unicorn_amd.native has
// loaded: its entry points are passed in by address (bind).
#include <torch/extension.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <map>
#include <stdexcept>
#include <string>

#include "../../include/unicorn_render.h"

namespace {

using at::Tensor;
using torch::autograd::collect_next_edges;
using torch::autograd::compute_requires_grad;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::set_history;
using torch::autograd::variable_list;

struct Api {
  decltype(&ur_last_error) last_error = nullptr;
  decltype(&ur_layer_norm_workspace_bytes) layer_norm_workspace_bytes = nullptr;
  decltype(&ur_layer_norm_forward) layer_norm_forward = nullptr;
  decltype(&ur_layer_norm_backward) layer_norm_backward = nullptr;
  decltype(&ur_route_workspace_bytes) route_workspace_bytes = nullptr;
  decltype(&ur_route_forward) route_forward = nullptr;
  decltype(&ur_route_backward) route_backward = nullptr;
  decltype(&ur_distill_workspace_bytes) distill_workspace_bytes = nullptr;
  decltype(&ur_distill_forward) distill_forward = nullptr;
  decltype(&ur_distill_backward) distill_backward = nullptr;
} api;

void bind(const std::map<std::string, uintptr_t>& address) {
#define UR_BIND(name) api.name = reinterpret_cast<decltype(api.name)>(address.at("ur_" #name));
  UR_BIND(last_error)
  UR_BIND(layer_norm_workspace_bytes) UR_BIND(layer_norm_forward) UR_BIND(layer_norm_backward)
  UR_BIND(route_workspace_bytes) UR_BIND(route_forward) UR_BIND(route_backward)
  UR_BIND(distill_workspace_bytes) UR_BIND(distill_forward) UR_BIND(distill_backward)
#undef UR_BIND
}

void check(int64_t rc, const char* what) {
  if (rc < 0) throw std::runtime_error(std::string(what) + " failed (" + std::to_string(rc) + "): " + api.last_error());
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return UR_F32;
    case at::kHalf: return UR_F16;
    case at::kBFloat16: return UR_BF16;
    default: throw std::invalid_argument("tensors must be float32, float16 or bfloat16");
  }
}

void same_device(const Tensor& t, const Tensor& other) {
  if (other.defined() && other.device() != t.device())
    throw std::invalid_argument("tensors must be on one device: " + t.device().str() + " and " + other.device().str());
}

// A tensor's numbers as they are in memory: a lazily negated view (`z.conj().imag`) is written out first.
Tensor stored(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// A tensor read as rows of its last dimension: as it lies where its rows are dense and evenly spaced without overlap (any
// stride between them), a contiguous copy otherwise.
struct Rows {
  Tensor t;
  int64_t rows, cols, stride;
  explicit Rows(const Tensor& x) : t(stored(x)), cols(x.size(-1)) {
    if (!t.is_contiguous()) {
      bool as_is = false;
      if (cols == 1 || t.stride(-1) == 1) {
        // one stride for all leading dimensions
        int64_t step = 0, count = 1;
        as_is = true;
        for (int64_t d = t.dim() - 2; d >= 0 && as_is; --d) {
          if (t.size(d) == 1) continue;
          if (count == 1) step = t.stride(d);
          else as_is = t.stride(d) == step * count;
          count *= t.size(d);
        }
        as_is = as_is && (count <= 1 || step >= cols);
        stride = count <= 1 ? cols : step;
      }
      if (!as_is) t = t.contiguous();
      if (as_is) {
        rows = cols ? t.numel() / cols : 0;
        return;
      }
    }
    rows = cols ? t.numel() / cols : 0;
    stride = cols;
  }
  const void* data() const { return t.const_data_ptr(); }
};

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* cptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
Tensor or_none(const std::optional<Tensor>& t) { return t.has_value() ? stored(*t) : Tensor(); }

// What the nodes know nothing of is refused.  A tangent of forward-mode differentiation would be dropped without a word.  A
// tracer records the allocation of a result but not the kernel that fills it: the trace would return uninitialised memory.
// Tensors of a function transform, and subclasses that dispatch for themselves, have no memory of their own to hand over.
void plain_inputs(std::initializer_list<Tensor> inputs) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  bool traced = torch::jit::tracer::isTracing();
  if (c10::impl::dispatch_mode_enabled())
    for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
      traced |= TorchDispatchModeTLS::get_mode(mode).has_value();
  if (traced) throw std::runtime_error("tracing is not supported by this operator: its kernels would not be in the trace");
  for (const Tensor& t : inputs) {
    if (!t.defined()) continue;
    const auto keys = t.key_set();
    if (keys.has_any(at::kFunctorchWrappedTensors) || keys.has(c10::DispatchKey::Batched) || keys.has(c10::DispatchKey::Python))
      throw std::runtime_error("function transforms (torch.func, batched gradients) and tensor subclasses with a dispatch of "
                               "their own are not supported by this operator");
    if (t._fw_grad(0).defined()) throw std::runtime_error("forward-mode differentiation is not supported by this operator");
  }
}

// A leaf's gradient accumulator belongs to the stream of the graph that made it and lives as long as that graph.  A captured
// backward that meets one of the default stream would make the default stream part of the capture, which ends the process.
void no_accumulator_of_default_stream(const Node& node) {
  for (const auto& edge : node.next_edges()) {
    if (!edge.function || !dynamic_cast<const torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
    const c10::Stream made_on = edge.function->input_metadata(0).stream();
    if (made_on.device_type() != c10::DeviceType::HIP && made_on.device_type() != c10::DeviceType::CUDA) continue;
    if (made_on.id() != 0 || c10::hip::getCurrentHIPStream(made_on.device_index()).id() == 0) continue;
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      throw std::runtime_error("a backward pass is being captured while a graph that was recorded on the default stream from the "
                               "same leaf is alive: drop that graph (its outputs) before the capture");
  }
}

// What a backward returns under create_graph: differentiating it again raises (the kernels are not recorded).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g.set_requires_grad(true);  // (or the error would not be attached)
  auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice an operator that can be "
                                                               "differentiated once", (int64_t)grads.size());
  return (*error)(std::move(grads));
}

// ---- layer norm -----------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> layer_norm_forward(const Tensor& x, const std::optional<Tensor>& weight,
                                              const std::optional<Tensor>& bias, double eps, bool need_stats) {
  const Tensor w = or_none(weight), b = or_none(bias);
  same_device(x, w);
  same_device(x, b);
  const c10::DeviceGuard guard(x.device());
  const Rows r(x);
  const int code = dtype_code(x.scalar_type());
  const int pcode = w.defined() ? dtype_code(w.scalar_type()) : b.defined() ? dtype_code(b.scalar_type()) : code;
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor stats = need_stats ? at::empty({2, r.rows}, x.options().dtype(at::kFloat)) : Tensor();
  if (r.rows) {
    const int64_t n = api.layer_norm_workspace_bytes(r.rows, r.cols, code, 0);
    check(n, "ur_layer_norm_workspace_bytes");
    const Tensor ws = workspace(n, x);
    float* mean = need_stats ? stats.mutable_data_ptr<float>() : nullptr;
    check(api.layer_norm_forward(r.data(), r.stride, cptr(w), cptr(b), code, pcode, r.rows, r.cols, (float)eps, ptr(y), mean,
                                 need_stats ? mean + r.rows : nullptr, ptr(ws), (size_t)n, stream_of(x)),
          "ur_layer_norm_forward");
  }
  return {y, stats};
}

// param_dtype: the type of the parameters and of their gradients
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& grad_y, const Tensor& x, const std::optional<Tensor>& weight,
                                                       at::ScalarType param_dtype, const Tensor& stats, bool need_x,
                                                       bool need_weight, bool need_bias) {
  const c10::DeviceGuard guard(x.device());
  const Rows r(x), g(grad_y);
  const Tensor w = or_none(weight);
  const int code = dtype_code(x.scalar_type()), pcode = dtype_code(param_dtype);
  Tensor gx, gw, gb;
  if (need_x) gx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (need_weight) gw = at::empty({r.cols}, x.options().dtype(param_dtype));
  if (need_bias) gb = at::empty({r.cols}, x.options().dtype(param_dtype));
  if (!r.rows) {
    if (need_weight) gw.zero_();
    if (need_bias) gb.zero_();
    return {gx, gw, gb};
  }
  const int64_t n = api.layer_norm_workspace_bytes(r.rows, r.cols, code, 1);
  check(n, "ur_layer_norm_workspace_bytes");
  const Tensor ws = workspace(n, x);
  const float* mean = stats.const_data_ptr<float>();
  check(api.layer_norm_backward(g.data(), g.stride, r.data(), r.stride, cptr(w), mean, mean + r.rows, code, pcode, r.rows, r.cols,
                                ptr(gx), ptr(gw), ptr(gb), ptr(ws), (size_t)n, stream_of(x)),
        "ur_layer_norm_backward");
  return {gx, gw, gb};
}

// A node keeps what its backward reads as SavedVariables (a change in place is noticed, a second backward without
// retain_graph raises) and the forward's own statistics, which nobody else sees, as they are.
struct LayerNormBackward : Node {
  SavedVariable x, weight;
  Tensor stats;
  at::ScalarType param_dtype = at::kFloat;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!grads[0].defined()) return out;
    plain_inputs({grads[0]});
    no_accumulator_of_default_stream(*this);
    const Tensor xs = x.unpack(), ws = weight.unpack();
    std::tie(out[0], out[1], out[2]) =
        layer_norm_backward(grads[0], xs, ws, param_dtype, stats, task_should_compute_output(0), task_should_compute_output(1),
                            task_should_compute_output(2));
    return once(std::move(out));
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    stats.reset();
  }
  std::string name() const override { return "LayerNormBackward"; }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  const Tensor w = or_none(weight), b = or_none(bias);
  plain_inputs({x, w, b});
  const bool record = compute_requires_grad(x, w, b);
  auto [y, stats] = layer_norm_forward(x, w, b, eps, record);
  if (record) {
    auto node = std::make_shared<LayerNormBackward>();
    node->set_next_edges(collect_next_edges(x, w, b));
    node->x = SavedVariable(x, false);
    node->weight = SavedVariable(w, false);
    node->param_dtype = (w.defined() ? w : b.defined() ? b : x).scalar_type();
    node->stats = stats;
    set_history(y, node);
  }
  return y;
}

// ---- routing --------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> route_forward(const Tensor& logits, const std::optional<Tensor>& bias, int64_t top_k,
                                                 int64_t score, int64_t groups, int64_t top_groups, int64_t group_score,
                                                 bool renormalize, double scale) {
  const Tensor b = or_none(bias);
  same_device(logits, b);
  const c10::DeviceGuard guard(logits.device());
  const Rows r(logits);
  auto shape = logits.sizes().vec();
  shape.back() = top_k;
  Tensor weights = at::empty(shape, logits.options().dtype(at::kFloat));
  Tensor indices = at::empty(shape, logits.options().dtype(at::kLong));
  Tensor counts = at::empty({r.cols}, logits.options().dtype(at::kInt));
  if (!r.rows) return {weights, indices, counts.zero_()};
  const int64_t n = api.route_workspace_bytes(r.rows, (int)r.cols);
  check(n, "ur_route_workspace_bytes");
  const Tensor ws = workspace(n, logits);
  check(api.route_forward(r.data(), r.stride, dtype_code(logits.scalar_type()), b.defined() ? b.const_data_ptr<float>() : nullptr,
                          r.rows, (int)r.cols, (int)top_k, (int)score, (int)groups, (int)top_groups, (int)group_score,
                          renormalize, (float)scale, weights.mutable_data_ptr<float>(), indices.mutable_data_ptr<int64_t>(),
                          counts.mutable_data_ptr<int32_t>(), ptr(ws), (size_t)n, stream_of(logits)),
        "ur_route_forward");
  return {weights, indices, counts};
}

Tensor route_backward(const Tensor& grad_weights, const Tensor& logits, const Tensor& weights, const Tensor& indices,
                      int64_t score, bool renormalize, double scale) {
  const c10::DeviceGuard guard(logits.device());
  const Rows r(logits);
  const Tensor g = stored(grad_weights).contiguous();
  Tensor grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  if (r.rows)
    check(api.route_backward(g.const_data_ptr<float>(), r.data(), r.stride, dtype_code(logits.scalar_type()), r.rows,
                             (int)r.cols, weights.const_data_ptr<float>(), indices.const_data_ptr<int64_t>(),
                             (int)indices.size(-1), (int)score, renormalize, (float)scale, ptr(grad), stream_of(logits)),
          "ur_route_backward");
  return grad;
}

struct RouteBackward : Node {
  SavedVariable logits, weights, indices;
  int64_t score = 0;
  bool renormalize = true;
  double scale = 1.0;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!grads[0].defined()) return out;
    plain_inputs({grads[0]});
    no_accumulator_of_default_stream(*this);
    out[0] = route_backward(grads[0], logits.unpack(), weights.unpack(shared_from_this()), indices.unpack(), score, renormalize,
                            scale);
    return once(std::move(out));
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits.reset_data();
    weights.reset_data();
    indices.reset_data();
  }
  std::string name() const override { return "RouteBackward"; }
};

std::tuple<Tensor, Tensor, Tensor> route(const Tensor& logits, const std::optional<Tensor>& bias, int64_t top_k, int64_t score,
                                         int64_t groups, int64_t top_groups, int64_t group_score, bool renormalize,
                                         double scale) {
  plain_inputs({logits, or_none(bias)});
  auto out = route_forward(logits, bias, top_k, score, groups, top_groups, group_score, renormalize, scale);
  if (compute_requires_grad(logits)) {
    auto node = std::make_shared<RouteBackward>();
    node->set_next_edges(collect_next_edges(logits));
    node->score = score;
    node->renormalize = renormalize;
    node->scale = scale;
    set_history(std::get<0>(out), node);
    node->logits = SavedVariable(logits, false);
    node->weights = SavedVariable(std::get<0>(out), true);
    node->indices = SavedVariable(std::get<1>(out), false);
  }
  return out;
}

// ---- distillation ---------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> distill_forward(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature,
                                           int64_t reduction, bool need_stats) {
  same_device(logits, teacher);
  same_device(logits, index);
  const c10::DeviceGuard guard(logits.device());
  const Rows r(logits);
  const bool per_row = reduction == UR_REDUCE_NONE;
  Tensor loss = at::empty(per_row ? logits.sizes().slice(0, logits.dim() - 1) : at::IntArrayRef(),
                          logits.options().dtype(at::kFloat));
  Tensor stats = need_stats ? at::empty({2 * r.rows + 1}, logits.options().dtype(at::kFloat)) : Tensor();
  if (!r.rows) return {per_row ? loss : loss.zero_(), stats};
  const int code = dtype_code(logits.scalar_type());
  const int64_t n = api.distill_workspace_bytes(r.rows, r.cols, code, (int)reduction);
  check(n, "ur_distill_workspace_bytes");
  const Tensor ws = workspace(n, logits);
  check(api.distill_forward(r.data(), r.stride, code, r.rows, r.cols, teacher.const_data_ptr(),
                            dtype_code(teacher.scalar_type()), index.const_data_ptr(), (int)index.element_size(),
                            (int)index.size(-1), temperature, (int)reduction, loss.mutable_data_ptr<float>(),
                            static_cast<float*>(ptr(stats)), ptr(ws), (size_t)n, stream_of(logits)),
        "ur_distill_forward");
  return {loss, stats};
}

Tensor distill_backward(const Tensor& grad_loss, const Tensor& logits, const Tensor& teacher, const Tensor& index,
                        double temperature, int64_t reduction, const Tensor& stats) {
  const c10::DeviceGuard guard(logits.device());
  const Rows r(logits);
  Tensor grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  if (!r.rows) return grad;
  const Tensor flat = stored(grad_loss), g = flat.dim() > 1 ? flat.reshape({-1}) : flat;
  check(api.distill_backward(g.const_data_ptr<float>(), g.dim() ? g.stride(0) : 0, r.data(), r.stride,
                             dtype_code(logits.scalar_type()), r.rows, r.cols, teacher.const_data_ptr(),
                             dtype_code(teacher.scalar_type()), index.const_data_ptr(), (int)index.element_size(),
                             (int)index.size(-1), temperature, (int)reduction, stats.const_data_ptr<float>(), ptr(grad),
                             stream_of(logits)),
        "ur_distill_backward");
  return grad;
}

struct DistillBackward : Node {
  SavedVariable logits, teacher, index;
  Tensor stats;
  double temperature = 1.0;
  int64_t reduction = UR_REDUCE_MEAN;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!grads[0].defined()) return out;
    plain_inputs({grads[0]});
    no_accumulator_of_default_stream(*this);
    const Tensor z = logits.unpack();
    out[0] = distill_backward(grads[0], z, teacher.unpack(), index.unpack(), temperature, reduction, stats);
    return once(std::move(out));
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits.reset_data();
    teacher.reset_data();
    index.reset_data();
    stats.reset();
  }
  std::string name() const override { return "DistillBackward"; }
};

Tensor distill(const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_index, double temperature,
               int64_t reduction) {
  plain_inputs({logits, teacher_logits, teacher_index});
  const Tensor teacher = stored(teacher_logits), index = stored(teacher_index);
  const bool record = compute_requires_grad(logits);
  auto [loss, stats] = distill_forward(logits, teacher, index, temperature, reduction, record);
  if (record) {
    auto node = std::make_shared<DistillBackward>();
    node->set_next_edges(collect_next_edges(logits));
    node->logits = SavedVariable(logits, false);
    node->teacher = SavedVariable(teacher, false);
    node->index = SavedVariable(index, false);
    node->stats = stats;
    node->temperature = temperature;
    node->reduction = reduction;
    set_history(loss, node);
  }
  return loss;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  using guard = py::call_guard<py::gil_scoped_release>;
  m.def("bind", &bind, "hand over the addresses of the library's entry points, {name: address}");
  m.def("layer_norm", &layer_norm, guard());
  m.def("layer_norm_forward", &layer_norm_forward, guard());
  m.def("route", &route, guard());
  m.def("distill", &distill, guard());
}
