// PyTorch side of expert routing and gradient clipping: argument checks, output and workspace allocation,
// autograd nodes and the calls of the C ABI, compiled instead of written in Python because the calls are
// short.  One gate of one row took 19 us through ctypes and a Python autograd.Function (forward and
// backward 119 us, of which the kernels are a few); a call is on a serving path.  No kernel lives here
// and no torch type crosses the C ABI.
//
// Errors: a broken contract raises RuntimeError, a failing entry point TBEError (a RuntimeError).
#include <pybind11/stl.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/jit/ir/ir.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/tbe_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

constexpr int64_t kMaxExperts = 1024, kMaxChoices = 32;

#define REQUIRE(cond, ...)                                             \
  do {                                                                 \
    if (!(cond)) throw std::runtime_error(c10::str(__VA_ARGS__));      \
  } while (0)

// A C entry point's failure; becomes TBEError on the way to Python.
struct EntryFailed : std::runtime_error {
  std::string entry, message;
  int64_t status;
  EntryFailed(const char* e, int64_t s)
      : std::runtime_error(c10::str(e, " failed with status ", s, ": ", tbe_last_error_string())),
        entry(e), message(tbe_last_error_string()), status(s) {}
};
void must(const char* entry, int64_t status) {
  if (status < 0) throw EntryFailed(entry, status);
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TBE_F32;
    case at::kHalf: return TBE_F16;
    case at::kDouble: return TBE_F64;
    case at::kBFloat16: return TBE_BF16;
    default: return -1;
  }
}
at::ScalarType weights_type(const Tensor& rows) { return rows.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

// A recorder sees the allocation of an output but not the kernel that fills it: what it records returns memory that
// nobody wrote.  Inside a Python autograd.Function (or a custom operator), which torch.jit.trace records as a whole and
// calls again, there is nothing to refuse.
bool jit_records_this() {
  if (!torch::jit::tracer::isTracing() || !at::tracer::impl::is_dispatch_enabled()) return false;
  // a Function gets its outputs when its forward has returned
  for (const torch::jit::Node* n : torch::jit::tracer::getTracingState()->graph->nodes())
    if (n->kind() == torch::jit::prim::PythonOp && n->outputs().empty()) return false;
  return true;
}
void refuse_recording() {
  REQUIRE(!jit_records_this() &&
              !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
          "expert routing and gradient clipping cannot be recorded (torch.jit.trace, make_fx, torch.export): wrap the "
          "call in an operator that the recorder keeps as a whole");
}

// Forward-mode differentiation keeps a tangent beside the tensor; what the kernels compute would come without one,
// which means a derivative of zero.  Tangents exist inside a dual_level() only; asking a view for one takes two locks
// (2 us for 40 tensors), so the level is asked first.
bool in_forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

void check_cuda(const char* name, const Tensor& t) {
  REQUIRE(!in_forward_mode() || !has_tangent(t), name, " carries a forward-mode tangent: there is no forward-mode derivative here");
  REQUIRE(t.defined() && t.is_cuda() && t.layout() == at::kStrided, name,
          " must be a CUDA tensor (this library has no CPU path)");
  REQUIRE(!t.is_neg(), name, " is a lazily negated view: call resolve_neg() on it");
}
void check_int32(const char* name, const Tensor& t) {
  check_cuda(name, t);
  REQUIRE(t.scalar_type() == at::kInt, name, " must have dtype torch.int32, got ", t.scalar_type());
}
void check_rows(const char* name, const Tensor& t) {
  check_cuda(name, t);
  REQUIRE(dtype_of(t) >= 0, name, " must be float16, bfloat16, float32 or float64, got ", t.scalar_type());
  REQUIRE(t.dim() == 2 && t.size(1) > 0, name, " must be two-dimensional with a non-empty row, got ", t.sizes());
}
// Rows whose elements are neighbours, with whatever stride between rows.
Tensor dense_rows(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int32_t* ints(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// An upstream gradient as the kernels read it: they see memory, not the negative bit that autograd may have set.
Tensor incoming(const Tensor& grad) {
  refuse_recording();
  REQUIRE(!in_forward_mode() || !has_tangent(grad), "the gradient carries a forward-mode tangent: there is no forward-mode derivative here");
  return grad.detach().resolve_neg();
}

// What a backward returns when its own graph is recorded: differentiating it again raises.
variable_list once(variable_list grads) {
  if (at::GradMode::is_enabled())
    for (Tensor& g : grads)
      if (g.defined()) {
        Tensor v = g.detach();
        v.set_requires_grad(true);
        auto node = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice an operator that is once differentiable", 1);
        g = (*node)({v})[0];
      }
  return grads;
}

// ---------------------------------------------------------------- gate
std::tuple<Tensor, Tensor> gate_forward(const Tensor& logits, int64_t k, bool renormalize) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const Tensor rows = dense_rows(logits);
  const int64_t N = rows.size(0), E = rows.size(1);
  Tensor weights = at::empty({N, k}, rows.options().dtype(weights_type(rows)));
  Tensor experts = at::empty({N, k}, rows.options().dtype(at::kInt));
  must("tbe_expert_gate", tbe_expert_gate(rows.data_ptr(), rows.stride(0), weights.data_ptr(), ints(experts), N, E, k,
                                          dtype_of(rows), renormalize, stream_of(rows)));
  return {weights, experts};
}

struct Gate : Function<Gate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, bool renormalize) {
    auto [weights, experts] = gate_forward(logits, k, renormalize);
    // the renormalized weights are all their gradient needs; the softmax over the whole row is redone
    ctx->save_for_backward({weights, experts, renormalize ? Tensor() : logits});
    ctx->saved_data["experts"] = logits.size(1);
    ctx->saved_data["dtype"] = static_cast<int64_t>(logits.scalar_type());
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({experts});
    return {weights, experts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor weights = saved[0].detach(), experts = saved[1];
    const c10::cuda::CUDAGuard guard(weights.device());
    const Tensor g = incoming(grads[0]).contiguous();
    const int64_t N = weights.size(0), k = weights.size(1), E = ctx->saved_data["experts"].toInt();
    Tensor out = at::empty({N, E}, weights.options().dtype(static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt())));
    const bool renormalize = !saved[2].defined();
    const Tensor rows = renormalize ? Tensor() : dense_rows(saved[2].detach());
    must("tbe_expert_gate_backward",
         tbe_expert_gate_backward(g.data_ptr(), data(rows), renormalize ? 0 : rows.stride(0), weights.data_ptr(),
                                  ints(experts), out.data_ptr(), N, E, k, dtype_of(out), renormalize, stream_of(out)));
    return once({out, Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> gate(const Tensor& logits, int64_t k, bool renormalize) {
  refuse_recording();
  check_rows("logits", logits);
  REQUIRE(logits.size(1) <= kMaxExperts, "logits must be [N, E] with E in 1..", kMaxExperts);
  REQUIRE(k >= 1 && k <= std::min(logits.size(1), kMaxChoices), "k must be in 1..min(E, ", kMaxChoices, "), got ", k);
  if (!logits.requires_grad() || !at::GradMode::is_enabled()) return gate_forward(logits, k, renormalize);
  auto out = Gate::apply(logits, k, renormalize);
  return {out[0], out[1]};
}

// ---------------------------------------------------------------- plan
std::tuple<Tensor, Tensor, Tensor> plan(const Tensor& choices, int64_t num_experts) {
  refuse_recording();
  check_int32("experts", choices);
  REQUIRE(choices.dim() == 2 && choices.size(1) > 0, "experts must be [N, k]");
  REQUIRE(num_experts >= 1 && num_experts <= kMaxExperts, "num_experts must be in 1..", kMaxExperts, ", got ", num_experts);
  const c10::cuda::CUDAGuard guard(choices.device());
  const Tensor experts = choices.contiguous();
  const int64_t M = experts.numel();
  Tensor offsets = at::empty({num_experts + 1}, experts.options());
  Tensor positions = at::empty(experts.sizes(), experts.options());
  Tensor order = at::empty({M}, experts.options());
  const int64_t bytes = tbe_expert_plan_workspace_bytes(M, num_experts);
  must("tbe_expert_plan_workspace_bytes", bytes);
  // a buffer of this call: calls on other streams and captured graphs have their own
  Tensor workspace = bytes ? at::empty({bytes / 4}, experts.options()) : Tensor();
  must("tbe_expert_plan", tbe_expert_plan(ints(experts), ints(offsets), ints(positions), ints(order), M, num_experts,
                                          data(workspace), bytes, stream_of(experts)));
  return {offsets, positions, order};
}

void check_plan(const Tensor& offsets, const Tensor& positions, const Tensor& rows) {
  check_int32("plan.offsets", offsets);
  check_int32("plan.positions", positions);
  REQUIRE(offsets.device() == rows.device() && positions.device() == rows.device(),
          "the plan and the rows are on different devices");
  REQUIRE(offsets.dim() == 1 && offsets.numel() >= 2 && offsets.is_contiguous(),
          "plan.offsets must be a contiguous [num_experts + 1]");
  REQUIRE(positions.dim() == 2 && positions.size(1) > 0 && positions.is_contiguous(),
          "plan.positions must be a contiguous [N, k]");
}

// ---------------------------------------------------------------- dispatch and combine
Tensor dispatch_rows(const Tensor& x, const Tensor& offsets, const Tensor& positions) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = dense_rows(x);
  const int64_t N = positions.size(0), k = positions.size(1), D = rows.size(1);
  Tensor y = at::empty({N * k, D}, rows.options());
  must("tbe_expert_dispatch", tbe_expert_dispatch(rows.data_ptr(), rows.stride(0), ints(positions), ints(offsets),
                                                  y.data_ptr(), N, k, D, offsets.numel() - 1, dtype_of(rows),
                                                  stream_of(rows)));
  return y;
}

Tensor combine_rows(const Tensor& y, const Tensor& offsets, const Tensor& positions, const Tensor& weights) {
  const c10::cuda::CUDAGuard guard(y.device());
  const Tensor rows = y.contiguous();
  const Tensor w = weights.defined() ? weights.contiguous() : Tensor();
  const int64_t N = positions.size(0), k = positions.size(1), D = rows.size(1);
  Tensor out = at::empty({N, D}, rows.options());
  must("tbe_expert_combine", tbe_expert_combine(rows.data_ptr(), ints(positions), ints(offsets), data(w), out.data_ptr(),
                                                N, k, D, offsets.numel() - 1, dtype_of(rows), stream_of(rows)));
  return out;
}

struct Dispatch : Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& offsets, const Tensor& positions) {
    ctx->save_for_backward({offsets, positions});
    ctx->set_materialize_grads(false);
    return dispatch_rows(x, offsets, positions);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    return once({combine_rows(incoming(grads[0]), saved[0], saved[1], Tensor()), Tensor(), Tensor()});
  }
};

struct Sum : Function<Sum> {  // combine without weights
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& offsets, const Tensor& positions) {
    ctx->save_for_backward({offsets, positions});
    ctx->set_materialize_grads(false);
    return combine_rows(y, offsets, positions, Tensor());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    return once({dispatch_rows(incoming(grads[0]), saved[0], saved[1]), Tensor(), Tensor()});
  }
};

struct Combine : Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor& offsets,
                        const Tensor& positions) {
    // the expert rows are only needed for the weights' gradient
    ctx->save_for_backward({weights.requires_grad() ? y : Tensor(), weights, offsets, positions});
    ctx->set_materialize_grads(false);
    return combine_rows(y, offsets, positions, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool need_y = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    if (!grads[0].defined() || (!need_y && !need_w)) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &offsets = saved[2], &positions = saved[3];
    const c10::cuda::CUDAGuard guard(offsets.device());
    const Tensor g = dense_rows(incoming(grads[0])), weights = saved[1].detach().contiguous();
    const Tensor y = need_w ? saved[0].detach().contiguous() : Tensor();
    const int64_t N = positions.size(0), k = positions.size(1), D = g.size(1);
    Tensor grad_y = need_y ? at::empty({N * k, D}, g.options()) : Tensor();
    Tensor grad_w = need_w ? at::empty({N, k}, weights.options()) : Tensor();
    must("tbe_expert_combine_backward",
         tbe_expert_combine_backward(g.data_ptr(), g.stride(0), data(y), ints(positions), ints(offsets), weights.data_ptr(),
                                     data(grad_y), data(grad_w), N, k, D, offsets.numel() - 1, dtype_of(g), stream_of(g)));
    return once({grad_y, grad_w, Tensor(), Tensor()});
  }
};

Tensor dispatch(const Tensor& x, const Tensor& offsets, const Tensor& positions) {
  refuse_recording();
  check_rows("x", x);
  check_plan(offsets, positions, x);
  REQUIRE(x.size(0) == positions.size(0), "x has ", x.size(0), " rows but the plan was made for ", positions.size(0));
  if (x.requires_grad() && at::GradMode::is_enabled()) return Dispatch::apply(x, offsets, positions);
  return dispatch_rows(x, offsets, positions);
}

Tensor combine(const Tensor& y, const Tensor& offsets, const Tensor& positions, const std::optional<Tensor>& weights) {
  refuse_recording();
  check_rows("y", y);
  check_plan(offsets, positions, y);
  const int64_t N = positions.size(0), k = positions.size(1);
  REQUIRE(y.size(0) == N * k, "y has ", y.size(0), " rows but the plan was made for ", N * k);
  const Tensor w = weights.value_or(Tensor());
  if (w.defined()) {
    check_cuda("weights", w);
    REQUIRE(w.scalar_type() == weights_type(y), "weights must have dtype ", weights_type(y), ", got ", w.scalar_type());
    REQUIRE(w.dim() == 2 && w.size(0) == N && w.size(1) == k, "weights must be [", N, ", ", k, "], got ", w.sizes());
    REQUIRE(w.device() == y.device(), "weights are on ", w.device(), " but y is on ", y.device());
  }
  if (at::GradMode::is_enabled()) {
    if (w.defined() && (y.requires_grad() || w.requires_grad())) return Combine::apply(y, w, offsets, positions);
    if (!w.defined() && y.requires_grad()) return Sum::apply(y, offsets, positions);
  }
  return combine_rows(y, offsets, positions, w);
}

// ---------------------------------------------------------------- gradients
struct List {
  std::vector<const void*> address;
  std::vector<int64_t> size;
  std::vector<int32_t> dtype;
  const Tensor* first = nullptr;

  explicit List(const std::vector<std::optional<Tensor>>& tensors) {
    address.reserve(tensors.size());
    size.reserve(tensors.size());
    dtype.reserve(tensors.size());
    const bool forward_mode = in_forward_mode();
    for (const auto& entry : tensors) {
      if (!entry.has_value()) continue;
      const Tensor& t = *entry;
      REQUIRE(!forward_mode || !has_tangent(t), "tensors carry a forward-mode tangent: there is no forward-mode derivative here");
      REQUIRE(t.defined() && t.is_cuda(), "tensors must be CUDA tensors (this library has no CPU path)");
      REQUIRE(t.layout() == at::kStrided && dtype_of(t) >= 0,
              "tensors must be dense float16, bfloat16, float32 or float64 tensors");
      REQUIRE(!t.is_neg(), "tensors must not be lazily negated views");
      REQUIRE(t.numel() == 0 || t.is_non_overlapping_and_dense(),
              "tensors must fill their memory without gaps or repeats (got strides ", t.strides(), " for ", t.sizes(), ")");
      if (!first) first = &t;
      REQUIRE(t.device() == first->device(), "tensors are on several devices");
      address.push_back(t.data_ptr());
      size.push_back(t.numel());
      dtype.push_back(dtype_of(t));
    }
  }
  int64_t count() const { return static_cast<int64_t>(address.size()); }
};

Tensor no_norm() {
  return at::zeros({}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA, c10::cuda::current_device()));
}

// a buffer of this call: calls on other streams and captured graphs have their own
Tensor norm_workspace(const List& list) {
  const int64_t bytes = tbe_grad_norm_workspace_bytes(list.count());
  must("tbe_grad_norm_workspace_bytes", bytes);
  return at::empty({bytes / 8}, at::TensorOptions().dtype(at::kDouble).device(list.first->device()));
}

Tensor grad_norm(const std::vector<std::optional<Tensor>>& tensors) {
  refuse_recording();
  const List list(tensors);
  if (!list.first) return no_norm();
  const c10::cuda::CUDAGuard guard(list.first->device());
  Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(list.first->device()));
  Tensor ws = norm_workspace(list);
  must("tbe_grad_norm", tbe_grad_norm(list.address.data(), list.size.data(), list.dtype.data(), list.count(),
                                      norm.data_ptr<float>(), ws.data_ptr(), ws.numel() * 8, stream_of(norm)));
  return norm;
}

bool same_order(const Tensor& a, const Tensor& b) {
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) != 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

Tensor clip_grad_norm(const std::vector<std::optional<Tensor>>& tensors, double max_norm, double eps,
                      const std::optional<std::vector<std::optional<Tensor>>>& out) {
  refuse_recording();
  REQUIRE(max_norm >= 0 && eps >= 0, "max_norm and eps must not be negative");
  const List list(tensors);
  if (out) REQUIRE(out->size() == tensors.size(), "out must have as many entries as tensors");
  if (!list.first) return no_norm();
  std::vector<void*> to;
  to.reserve(list.address.size());
  const bool forward_mode = in_forward_mode();
  for (size_t i = 0; i < tensors.size(); ++i) {
    if (!tensors[i].has_value()) continue;
    const Tensor& t = *tensors[i];
    if (out) {
      const auto& o = (*out)[i];
      REQUIRE(!forward_mode || !o.has_value() || !has_tangent(*o),
              "out carries a forward-mode tangent: there is no forward-mode derivative here");
      REQUIRE(o.has_value() && o->defined() && o->layout() == at::kStrided && !o->is_neg() && o->device() == t.device() &&
                  o->scalar_type() == t.scalar_type() && o->sizes() == t.sizes() && same_order(*o, t),
              "out must match tensors in device, type, shape and strides");
      to.push_back(o->data_ptr());
    } else {
      to.push_back(t.data_ptr());
    }
  }
  const c10::cuda::CUDAGuard guard(list.first->device());
  Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(list.first->device()));
  Tensor ws = norm_workspace(list);
  // autograd notices that a saved tensor is written to (an inference tensor outside inference mode is refused here)
  for (size_t i = 0; i < tensors.size(); ++i)
    if (tensors[i].has_value()) (out ? *(*out)[i] : *tensors[i]).unsafeGetTensorImpl()->bump_version();
  must("tbe_grad_clip", tbe_grad_clip(list.address.data(), to.data(), list.size.data(), list.dtype.data(), list.count(),
                                      max_norm, eps, norm.data_ptr<float>(), ws.data_ptr(), ws.numel() * 8,
                                      stream_of(norm)));
  return norm;
}

}  // namespace

PYBIND11_MODULE(_torch_glue, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const EntryFailed& e) {
      const py::object type = py::module_::import("sparse_ads_baselines_b200._lib").attr("TBEError");
      const py::object error = type(e.entry, e.status, e.message);
      PyErr_SetObject(type.ptr(), error.ptr());
    }
  });
  using nogil = py::call_guard<py::gil_scoped_release>;
  m.def("gate", &gate, nogil());
  m.def("plan", &plan, nogil());
  m.def("dispatch", &dispatch, nogil());
  m.def("combine", &combine, nogil());
  m.def("grad_norm", &grad_norm, nogil());
  m.def("clip_grad_norm", &clip_grad_norm, nogil());
}
