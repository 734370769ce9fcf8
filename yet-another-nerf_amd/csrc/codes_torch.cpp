// The learned codes' autograd nodes: lookup, its gradient and dropout as torch operations over the C ABI's entry points.
//
// A call of these is short next to what Python adds around it. With the nodes written in Python (torch.autograd.Function
// over ctypes, as the MLP's and the compositing's are) a forward and a backward of one 32-element row took 78 us of the
// host, with them here 41; the kernels need 6. The engine runs a backward on a thread of its own, and what remains is mostly
// the two hand-overs between the threads. A lookup without a gradient: 9 us in Python, 5 here. No kernels in this file: the
// entry points of libyanerf_hip.so come in as addresses (_C.py).
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/Functions.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <limits>
#include <optional>
#include <string>

#include "../../include/yanerf_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::variable_list;

namespace {

struct {
  decltype(&yanerf_last_error) last_error;
  decltype(&yanerf_dropout) dropout;
  decltype(&yanerf_embedding_forward) lookup;
  decltype(&yanerf_embedding_bwd_workspace_bytes) workspace;
  decltype(&yanerf_embedding_backward) gradient;
} api;

void bind(uintptr_t last_error, uintptr_t dropout, uintptr_t lookup, uintptr_t workspace, uintptr_t gradient) {
  api = {(decltype(api.last_error))last_error, (decltype(api.dropout))dropout, (decltype(api.lookup))lookup,
         (decltype(api.workspace))workspace, (decltype(api.gradient))gradient};
}

void done(int status, const char* what) {
  if (status) throw std::runtime_error(std::string(what) + " failed: " + api.last_error());
}

int type_of(at::ScalarType t) {
  return t == at::kFloat ? YANERF_TYPE_F32 : t == at::kBFloat16 ? YANERF_TYPE_BF16 : t == at::kHalf ? YANERF_TYPE_F16 : -1;
}
at::ScalarType scalar_of(int type) {
  return type == YANERF_TYPE_F32 ? at::kFloat : type == YANERF_TYPE_BF16 ? at::kBFloat16 : at::kHalf;
}

// A tensor's device made current for a launch, and its current stream
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream((void*)c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// What a backward needs to draw its forward's mask again: (seed, offset), or the offset that the forward's kernel read
// from rng_base, kept in `used`, as the base may have moved on by then
struct Mask {
  double p = 0.0;
  uint64_t seed = 0, offset = 0;
  std::optional<Tensor> base;
  Tensor used;

  void check(const char* what, const Tensor& like) const {
    if (!(p >= 0.0 && p <= 1.0))
      throw py::value_error(std::string(what) + ": dropout probability " + std::to_string(p) + " is not in [0, 1]");
    if (!base) return;
    if (!base->is_cuda() || base->device() != like.device() || base->numel() != 1 || base->is_neg() ||
        (base->scalar_type() != at::kLong && base->scalar_type() != at::kUInt64))
      throw py::value_error(std::string(what) + ": rng_base must be one int64 / uint64 element on " +
                            like.device().str());
  }
  const uint64_t* base_ptr() const { return base && p > 0.0 ? (const uint64_t*)base->data_ptr() : nullptr; }
  // for the forward of a call that has a backward
  void keep() {
    if (base && p > 0.0) used = at::empty({1}, base->options());
  }
  uint64_t* used_ptr() const { return used.defined() ? (uint64_t*)used.data_ptr() : nullptr; }
  uint64_t again_offset() const { return used.defined() ? 0 : offset; }
};

// These calls are no operators of torch's dispatcher: one that records operators sees nothing of them but the allocation of
// their outputs, and a replay would return memory that nobody wrote. Modes that only watch stay allowed.
void refuse_recording(const char* what) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  const char* by = nullptr;
  if (torch::jit::tracer::isTracing()) by = "torch.jit.trace";
  else if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) by = "a pre-dispatch trace";
  else if (TorchDispatchModeTLS::any_modes_set()) {
    if (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY)) by = "make_fx";
    else if (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE)) by = "a fake tensor mode";
    else if (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL)) by = "a functionalization mode";
  }
  if (by) throw std::runtime_error(std::string(what) + ": cannot be recorded by " + by);
}

void refuse_tangent(const char* what, const Tensor& t) {
  if (t._fw_grad(/*level=*/0).defined())
    throw std::runtime_error(std::string(what) + ": forward-mode differentiation is not supported");
}
void refuse_graph(const char* what, const Tensor& g) {
  refuse_tangent(what, g);
  if (at::GradMode::is_enabled() && g.requires_grad())
    throw std::runtime_error(std::string(what) + ": a gradient of its gradient (create_graph=True) is not supported");
}

// Its values in memory: contiguous() hands a contiguous view whose values are the negated memory back as it is
Tensor resolved(const Tensor& t) { return t.resolve_neg().contiguous(); }

// What a backward may read of the gradient it is given: the engine has compared it with the output, a direct call of the node
// has not
struct Output {
  int64_t numel = 0;
  at::ScalarType type = at::kFloat;
  c10::Device device = c10::Device(c10::kCUDA);
  explicit Output(const Tensor& y) : numel(y.numel()), type(y.scalar_type()), device(y.device()) {}
  Output() = default;
  void check(const char* what, const Tensor& g) const {
    if (g.device() != device || g.scalar_type() != type || g.numel() != numel)
      throw std::runtime_error(std::string(what) + ": the gradient differs from the output in device, type or size");
  }
};

// ------------------------------------------------------------------------------------------ dropout
Tensor run_dropout(const Tensor& x, const Mask& m, uint64_t offset, const uint64_t* base, uint64_t* used) {
  Tensor y = at::empty(x.sizes(), x.options());
  On on(x);
  done(api.dropout(x.data_ptr(), type_of(x.scalar_type()), x.numel(), m.p, m.seed, offset, base, used, y.data_ptr(),
                   on.stream),
       "yanerf_dropout");
  return y;
}

struct DropoutBackward : Node {
  Mask mask;
  Output output;
  std::string name() const override { return "YanerfDropoutBackward"; }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
    refuse_recording("dropout");
    refuse_graph("dropout", grads[0]);
    output.check("dropout", grads[0]);
    at::NoGradGuard no_grad;
    return {run_dropout(resolved(grads[0]), mask, mask.again_offset(), mask.used_ptr(), nullptr)};
  }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const std::optional<Tensor>& rng_base) {
  refuse_recording("dropout");
  if (type_of(x.scalar_type()) < 0)
    throw py::type_error(std::string("dropout: element type ") + c10::toString(x.scalar_type()) +
                         " is not supported (float32, bfloat16, float16)");
  Mask m{p, seed, offset, rng_base, Tensor()};
  m.check("dropout", x);
  refuse_tangent("dropout", x);
  const bool graph = at::GradMode::is_enabled() && x.requires_grad();
  if (graph) m.keep();
  Tensor y;
  {
    at::NoGradGuard no_grad;
    y = run_dropout(resolved(x), m, m.offset, m.base_ptr(), m.used_ptr());
  }
  if (graph) {
    auto node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
    node->mask = m;
    node->output = Output(y);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ------------------------------------------------------------------------------------------ lookup
struct EmbeddingBackward : Node {
  torch::autograd::SavedVariable ids;
  Mask mask;
  Output output;
  int64_t V = 0, D = 0, pad = -1;
  double scale = 1.0;
  at::ScalarType type = at::kFloat;
  std::string name() const override { return "YanerfEmbeddingBackward"; }
  void release_variables() override { ids.reset_data(); }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
    refuse_recording("embedding");
    refuse_graph("embedding", grads[0]);
    output.check("embedding", grads[0]);
    at::NoGradGuard no_grad;
    const Tensor i = resolved(ids.unpack()), g = resolved(grads[0]);
    // hooks of saved tensors may hand back another tensor than was saved
    if (i.device() != output.device || (i.scalar_type() != at::kLong && i.scalar_type() != at::kInt) ||
        i.numel() * D != output.numel)
      throw std::runtime_error("embedding: the saved ids came back with another device, type or size");
    const int64_t N = i.numel(), bytes = api.workspace(N, V, D);
    if (bytes < 0) done(1, "yanerf_embedding_bwd_workspace_bytes");
    Tensor grad = at::empty({V, D}, g.options().dtype(type));
    Tensor ws;
    if (bytes) ws = at::empty({bytes}, g.options().dtype(at::kByte));
    On on(g);
    done(api.gradient(g.data_ptr(), type_of(g.scalar_type()), i.data_ptr(), (int)i.element_size(), N, V, D, pad, scale,
                      mask.p, mask.seed, mask.again_offset(), mask.used_ptr(), grad.data_ptr(), type_of(type),
                      bytes ? ws.data_ptr() : nullptr, on.stream),
         "yanerf_embedding_backward");
    return {grad};
  }
};

// out_type: -1 for the table's; flag: address of the device's flag of ids outside their table, or 0
Tensor embedding(const Tensor& table, const Tensor& ids_in, double scale, std::optional<int64_t> padding_idx, double p,
                 uint64_t seed, uint64_t offset, const std::optional<Tensor>& rng_base, int out_type, uintptr_t flag) {
  refuse_recording("embedding");
  if (table.dim() != 2)
    throw py::value_error("embedding: the table must be [V, D], got " + std::to_string(table.dim()) + " dimensions");
  const int type = type_of(table.scalar_type());
  if (type < 0)
    throw py::type_error(std::string("embedding: element type ") + c10::toString(table.scalar_type()) +
                         " is not supported (float32, bfloat16, float16)");
  if (ids_in.scalar_type() != at::kLong && ids_in.scalar_type() != at::kInt)
    throw py::type_error(std::string("embedding: ids must be int32 or int64, got ") +
                         c10::toString(ids_in.scalar_type()));
  if (ids_in.device() != table.device())
    throw std::runtime_error("embedding: ids on " + ids_in.device().str() + ", table on " + table.device().str());
  const int64_t V = table.size(0), D = table.size(1);
  if (V == 0 && ids_in.numel()) throw py::index_error("embedding: ids into an empty table");
  int64_t pad = -1;
  if (padding_idx) {
    if (*padding_idx < -V || *padding_idx >= V)
      throw py::value_error("embedding: padding_idx " + std::to_string(*padding_idx) + " is outside a table of " +
                            std::to_string(V) + " rows");
    pad = *padding_idx < 0 ? *padding_idx + V : *padding_idx;
  }
  if (!std::isfinite(scale)) throw py::value_error("embedding: scale is not finite");
  Mask m{p, seed, offset, rng_base, Tensor()};
  m.check("embedding", table);
  const double f = p < 1.0 ? scale / (1.0 - p) : 0.0;
  if (f != 0.0 && !(std::fabs(f) >= std::numeric_limits<float>::min() && std::fabs(f) <= std::numeric_limits<float>::max()))
    throw py::value_error("embedding: the factor scale / (1 - dropout) is outside the range of fp32");
  refuse_tangent("embedding", table);
  const bool graph = at::GradMode::is_enabled() && table.requires_grad();
  if (graph) m.keep();
  Tensor out, ids;
  {
    at::NoGradGuard no_grad;
    const Tensor t = D > 1 && table.stride(1) != 1 ? resolved(table) : table.resolve_neg();
    ids = resolved(ids_in);
    c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(D);
    out = at::empty(shape, t.options().dtype(out_type < 0 ? table.scalar_type() : scalar_of(out_type)));
    On on(t);
    done(api.lookup(t.data_ptr(), type, t.stride(0), ids.data_ptr(), (int)ids.element_size(), ids.numel(), V, D, scale,
                    m.p, m.seed, m.offset, m.base_ptr(), m.used_ptr(), out.data_ptr(), out_type < 0 ? type : out_type,
                    (int*)flag, on.stream),
         "yanerf_embedding_forward");
  }
  if (graph) {
    auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
    node->ids = torch::autograd::SavedVariable(ids, /*is_output=*/false);
    node->mask = m;
    node->output = Output(out);
    node->V = V;
    node->D = D;
    node->pad = pad;
    node->scale = scale;
    node->type = table.scalar_type();
    node->set_next_edges(torch::autograd::collect_next_edges(table));
    torch::autograd::set_history(out, node);
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(_codes_torch, m) {
  m.def("build_id", [] { return YANERF_SRC_SHA; });
  m.def("torch_version", [] { return YANERF_TORCH_VERSION; });
  m.def("bind", &bind);
  m.def("refuse_recording", &refuse_recording);
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
  m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
}
