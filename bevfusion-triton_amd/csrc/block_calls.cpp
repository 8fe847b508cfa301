// block_calls.cpp -- the block operators as functions of tensors, and their
// gradients as nodes of torch's autograd graph, in C++ beside the C ABI that
// they call.  Arguments are checked in Python (block.py).
//
// A call on a few tokens is bound by the host, and so is a training step on a
// few thousand: the backward pass runs on the autograd engine's thread, and in
// Python the interpreter's objects go back and forth between two cores.  us of a
// step on a few tokens by Python functions over ctypes and by this: residual_norm
// with all its operands 143 and 87, gated_activation 85 and 44, checkpoint_linear
// 165 and 98 (torch's own linear 102); of a call without gradients 12.5 and 9.1,
// 7.7 and 5.8, linear_int8 10.7 and 7.6.
//
// What is not followed by a gradient's node is followed by a Python function
// (traces, tangents), which calls the *_forward and *_backward here.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>

#include "bevpool.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// ---- calls -----------------------------------------------------------------

struct CallError : public std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject *call_error = nullptr;  // what Python sees of it
void check(int status, const char *what) {
  if (status != BEVPOOL_OK)
    throw CallError(std::string(what) + " failed (status " + std::to_string(status) +
                             "): " + bevpool_last_error());
}
int code_of(at::ScalarType type) {
  return type == at::kFloat ? BEVPOOL_F32 : type == at::kHalf ? BEVPOOL_F16 : BEVPOOL_BF16;
}
void *stream() { return c10::hip::getCurrentHIPStream().stream(); }  // of the current device
void *at_of(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t row_of(const Tensor &t) { return t.defined() ? t.stride(0) : 0; }
Tensor given(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }
std::vector<Maybe> maybe(const variable_list &tensors) {
  std::vector<Maybe> out;
  for (const Tensor &t : tensors) out.push_back(maybe(t));
  return out;
}
Tensor bytes(const Tensor &like, size_t n) {
  return at::empty({int64_t(n)}, like.options().dtype(at::kByte));
}

// room for an 8-bit checkpoint of rows
Tensor kept_rows(const Tensor &x, int64_t rows, int64_t width, int copies = 1) {
  return at::empty({rows, copies * bevpool_checkpoint_pitch(int(width))},
                   x.options().dtype(at::kByte));
}

// What a backward pass reads.  Saved tensors come back by way of hooks, and
// gradients from whoever calls a node: of another size, type or place than the
// forward's they are refused, before a kernel reads past them; in another layout
// they are copied.  (1 us of a step on few tokens.)
struct Given {
  at::Device device;  // that of the gradients
  explicit Given(const Tensor &grad) : device(grad.device()) {
    TORCH_CHECK(grad.is_cuda(), "a gradient is not on the GPU");
  }
  Tensor fits(const Tensor &t, at::ScalarType type, at::IntArrayRef sizes, const char *what) const {
    TORCH_CHECK(t.device() == device && t.scalar_type() == type && t.sizes() == sizes, what,
                " of a backward pass is not the forward's: ", t.scalar_type(), " ", t.sizes(),
                " on ", t.device(), " for ", type, " ", sizes, " on ", device);
    return t;
  }
  // (rows have unit stride along them)
  Tensor rows(const Tensor &t, at::ScalarType type, int64_t n, int64_t width, const char *what) const {
    if (!t.defined()) return t;
    fits(t, type, {n, width}, what);
    return t.stride(1) == 1 || width == 1 ? t : t.contiguous();
  }
  Tensor grad(const Tensor &t, at::ScalarType type, int64_t n, int64_t width) const {
    return t.defined() && t.scalar_type() != type ? rows(t.to(type), type, n, width, "a gradient")
                                                  : rows(t, type, n, width, "a gradient");
  }
  Tensor vector(const Tensor &t, at::ScalarType type, int64_t width, const char *what) const {
    return t.defined() ? fits(t, type, {width}, what).contiguous() : t;
  }
  // (from a multiple of 16 bytes, as an allocation is)
  Tensor kept(const Tensor &t, int64_t n, int64_t width, int copies = 1) const {
    if (!t.defined()) return t;
    fits(t, at::kByte, {n, copies * bevpool_checkpoint_pitch(int(width))}, "a checkpoint");
    const bool lies = t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return lies ? t : t.clone(at::MemoryFormat::Contiguous);
  }
};

// Sum and normed of rows, and the checkpoints of x and update.
variable_list residual_forward(const Tensor &x, const Tensor &update, const Tensor &update_weight,
                               const Tensor &scale, const Tensor &gate, const Tensor &weight,
                               at::ScalarType type, double eps, bool keep) {
  const c10::DeviceGuard device(x.device());
  const int64_t rows = x.size(0), width = x.size(1);
  Tensor sum, normed, x_kept, update_kept;
  if (update.defined()) sum = at::empty({rows, width}, x.options());
  if (weight.defined()) normed = at::empty({rows, width}, x.options().dtype(type));
  // (the norm before the next block alone needs x for its gradient)
  if (keep && weight.defined()) x_kept = kept_rows(x, rows, width);
  if (keep && update.defined()) update_kept = kept_rows(x, rows, width);
  check(bevpool_residual_norm_forward(
            at_of(x), row_of(x), code_of(x.scalar_type()), at_of(update), row_of(update),
            at_of(update_weight), at_of(scale), at_of(gate), row_of(gate),
            gate.defined() ? gate.size(0) : 0, at_of(weight), code_of(type), rows, int(width),
            float(eps), at_of(sum), at_of(normed), at_of(x_kept), at_of(update_kept), stream()),
        "bevpool_residual_norm_forward");
  return {sum, normed, x_kept, update_kept};
}

struct Residual {
  int64_t rows, width;
  at::ScalarType x_type, type;
  double eps;
  bool kept, has_update;
};
// Gradients of x, update, update_weight, scale, gate and weight.
variable_list residual_backward(const Residual &R, Tensor dsum, Tensor dnormed, Tensor x,
                                Tensor update, Tensor update_weight, Tensor scale, Tensor gate,
                                Tensor weight) {
  if (!dsum.defined() && !dnormed.defined()) return variable_list(6);
  const Given in(dsum.defined() ? dsum : dnormed);
  const c10::DeviceGuard device(in.device);
  const auto options = (dsum.defined() ? dsum : dnormed).options();
  dsum = in.grad(dsum, R.x_type, R.rows, R.width);
  dnormed = in.grad(dnormed, R.type, R.rows, R.width);
  x = R.kept ? in.kept(x, R.rows, R.width) : in.rows(x, R.x_type, R.rows, R.width, "x");
  update = R.kept ? in.kept(update, R.rows, R.width)
                  : in.rows(update, R.type, R.rows, R.width, "update");
  update_weight = in.vector(update_weight, R.type, R.width, "update_weight");
  scale = in.vector(scale, R.type, R.width, "scale");
  weight = in.vector(weight, R.type, R.width, "weight");
  if (gate.defined()) gate = in.rows(gate, R.type, gate.size(0), R.width, "gate");
  const auto wide = options.dtype(R.x_type), own = options.dtype(R.type);
  Tensor dweight;
  if (weight.defined()) dweight = dnormed.defined() ? at::empty({R.width}, own) : at::zeros_like(weight);
  if (!dnormed.defined()) {
    weight = Tensor();
    x = Tensor();
  }
  Tensor dx = at::empty({R.rows, R.width}, wide), dupdate, dupdate_weight, dscale, dgate;
  if (R.has_update) dupdate = at::empty({R.rows, R.width}, own);
  if (update_weight.defined()) dupdate_weight = at::empty({R.width}, own);
  if (scale.defined()) dscale = at::empty({R.width}, own);
  const int64_t gate_rows = gate.defined() ? gate.size(0) : 0;
  // (no kernel writes the sums of no rows)
  if (gate.defined()) dgate = R.rows ? at::empty({gate_rows, R.width}, own) : at::zeros_like(gate);
  const int width = int(R.width), x_code = code_of(R.x_type);
  const size_t need =
      bevpool_residual_norm_backward_scratch_bytes(R.rows, width, gate_rows, x_code, R.kept);
  const Tensor scratch = bytes(dx, need);
  check(bevpool_residual_norm_backward(
            at_of(x), row_of(x), x_code, at_of(update), row_of(update), at_of(update_weight),
            at_of(scale), at_of(gate), row_of(gate), gate_rows, at_of(weight), R.kept, at_of(dsum),
            row_of(dsum), at_of(dnormed), row_of(dnormed), code_of(R.type), R.rows, width,
            float(R.eps), at_of(dx), at_of(dupdate), at_of(dgate), at_of(dupdate_weight),
            at_of(dscale), weight.defined() ? at_of(dweight) : nullptr, at_of(scratch), need,
            stream()),
        "bevpool_residual_norm_backward");
  return {dx, dupdate, dupdate_weight, dscale, dgate, dweight};
}

// The activation and the checkpoint.
variable_list gated_forward(const Tensor &x, int kind, bool keep) {
  const c10::DeviceGuard device(x.device());
  const int64_t rows = x.size(0), width = x.size(1) / 2;
  const Tensor out = at::empty({rows, width}, x.options());
  Tensor kept;
  if (keep) kept = kept_rows(x, rows, width, 2);
  check(bevpool_gated_forward(at_of(x), row_of(x), code_of(x.scalar_type()), rows, int(width), kind,
                              at_of(out), at_of(kept), stream()),
        "bevpool_gated_forward");
  return {out, kept};
}

struct Gated {
  int64_t rows, width;
  at::ScalarType type;
  int kind;
  bool kept;
};
variable_list gated_backward(const Gated &G, Tensor dout, Tensor x) {
  if (!dout.defined()) return variable_list(1);
  const Given in(dout);
  const c10::DeviceGuard device(in.device);
  dout = in.grad(dout, G.type, G.rows, G.width);
  x = G.kept ? in.kept(x, G.rows, G.width, 2)
             : in.rows(x, G.type, G.rows, 2 * G.width, "x");
  const Tensor dx = at::empty({G.rows, 2 * G.width}, dout.options());
  check(bevpool_gated_backward(at_of(x), row_of(x), G.kept, at_of(dout), row_of(dout),
                               code_of(G.type), G.rows, int(G.width), G.kind, at_of(dx), stream()),
        "bevpool_gated_backward");
  return {dx};
}

Tensor pack(const Tensor &x) {
  const c10::DeviceGuard device(x.device());
  const Tensor kept = kept_rows(x, x.size(0), x.size(1));
  check(bevpool_checkpoint_pack(at_of(x), row_of(x), code_of(x.scalar_type()), x.size(0),
                                int(x.size(1)), at_of(kept), stream()),
        "bevpool_checkpoint_pack");
  return kept;
}

Tensor linear8(const Tensor &x, const Tensor &codes, int64_t row, const Tensor &scales,
               const Tensor &bias) {
  const c10::DeviceGuard device(x.device());
  const int64_t rows = x.size(0), channels = scales.size(0);
  const int width = int(x.size(1));
  const Tensor y = at::empty({rows, channels}, x.options());
  const size_t need = bevpool_linear8_scratch_bytes(rows, width);
  const Tensor scratch = bytes(x, need);
  check(bevpool_linear8(at_of(x), row_of(x), code_of(x.scalar_type()), at_of(codes), row,
                        at_of(scales), at_of(bias), rows, width, channels, at_of(y), at_of(scratch),
                        need, stream()),
        "bevpool_linear8");
  return y;
}

struct Linear {
  int64_t rows, width;
  at::ScalarType type;
  bool direct;  // the weight's gradient from the checkpoint itself
};
// Gradients of x, weight and bias, those that are needed.
variable_list linear_backward(const Linear &A, Tensor dy, Tensor kept, const Tensor &weight,
                              bool need_x, bool need_weight, bool need_bias) {
  variable_list grads(3);
  if (!dy.defined()) return grads;
  const Given in(dy);
  const c10::DeviceGuard device(in.device);
  in.fits(weight, A.type, {weight.dim() ? weight.size(0) : 0, A.width}, "weight");
  const int n = int(weight.size(0)), k = int(A.width), code = code_of(A.type);
  if (dy.scalar_type() != A.type) dy = dy.to(A.type);
  in.fits(dy, A.type, {A.rows, n}, "a gradient");  // (the library takes any layout)
  kept = in.kept(kept, A.rows, A.width);
  if (need_x) grads[0] = dy.mm(weight);
  if (need_weight && A.direct && A.rows) {
    Tensor rows = dy;
    if (dy.stride(1) != 1 || dy.stride(0) % 8 || reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 ||
        dy.stride(0) >= (1 << 24))
      rows = dy.clone(at::MemoryFormat::Contiguous);
    grads[1] = at::empty({n, k}, dy.options());
    const size_t need = bevpool_checkpoint_weight_grad_scratch_bytes(A.rows, n, k);
    const Tensor scratch = bytes(dy, need);
    check(bevpool_checkpoint_weight_grad(at_of(rows), row_of(rows), at_of(kept), code, A.rows, n, k,
                                         at_of(grads[1]), at_of(scratch), need, stream()),
          "bevpool_checkpoint_weight_grad");
  } else if (need_weight) {
    const Tensor x = at::empty({A.rows, A.width}, dy.options());
    check(bevpool_checkpoint_unpack(at_of(kept), code, A.rows, k, at_of(x), stream()),
          "bevpool_checkpoint_unpack");
    grads[1] = dy.t().mm(x);
  }
  if (need_bias) grads[2] = at::empty({n}, dy.options());
  if (need_bias && n > 0) {  // (the sums refuse rows of nothing)
    const Tensor rows = in.rows(dy, A.type, A.rows, n, "a gradient");
    const size_t need = bevpool_column_sums_scratch_bytes(n);
    const Tensor scratch = bytes(dy, need);
    check(bevpool_column_sums(at_of(rows), row_of(rows), code, A.rows, n, at_of(grads[2]),
                              at_of(scratch), need, stream()),
          "bevpool_column_sums");
  }
  return grads;
}

// ---- nodes -----------------------------------------------------------------

// A refusal as Python's own error: the only ones whose type the engine carries to
// the thread that waits for it.
[[noreturn]] void raise(const CallError &refusal) {
  const pybind11::gil_scoped_acquire held;
  PyErr_SetString(call_error ? call_error : PyExc_RuntimeError, refusal.what());
  python_error error;
  error.persist();
  throw error;
}

// A node keeps tensors; its body gets them back.  Gradients are no functions of
// the graph's: a second derivative is refused.
template <int kSaved>
struct Recorded : public Node {
  SavedVariable saved[kSaved];
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable &s : saved) s.reset_data();
  }
  virtual variable_list body(variable_list &&grads, const variable_list &kept) = 0;
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list kept;
    kept.reserve(kSaved);
    for (const SavedVariable &s : saved) kept.push_back(s.unpack());
    const bool followed = at::GradMode::is_enabled();
    variable_list out;
    try {
      const at::NoGradGuard none;
      out = body(std::move(grads), kept);
    } catch (const CallError &refusal) {
      raise(refusal);
    }
    if (!followed) return out;
    for (Tensor &t : out)
      if (t.defined()) t = t.detach().set_requires_grad(true);
    torch::autograd::DelayedError refusal(
        "a second derivative of " + name() + " was asked for, which it does not have",
        int64_t(out.size()));
    return refusal.apply(std::move(out));
  }
};
template <typename N, typename... Inputs>
std::shared_ptr<N> node_of(const Inputs &...inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

struct ResidualNode : public Recorded<6> {
  Residual call;
  std::string name() const override { return "residual_norm"; }
  variable_list body(variable_list &&g, const variable_list &s) override {
    return residual_backward(call, g[0], g[1], s[0], s[1], s[2], s[3], s[4], s[5]);
  }
};
struct GatedNode : public Recorded<1> {
  Gated call;
  std::string name() const override { return "gated_activation"; }
  variable_list body(variable_list &&g, const variable_list &s) override {
    return gated_backward(call, g[0], s[0]);
  }
};
struct LinearNode : public Recorded<2> {
  Linear call;
  std::string name() const override { return "checkpoint_linear"; }
  variable_list body(variable_list &&g, const variable_list &s) override {
    return linear_backward(call, g[0], s[0], s[1], task_should_compute_output(0),
                           task_should_compute_output(1), task_should_compute_output(2));
  }
};

// ---- calls with their nodes, and what Python calls ------------------------------------------------------------

std::pair<Maybe, Maybe> residual_norm(const Tensor &x, const Maybe &update, const Maybe &update_weight,
                                      const Maybe &scale, const Maybe &gate, const Maybe &weight,
                                      at::ScalarType type, double eps, bool keep, bool follow) {
  const Tensor u = given(update), uw = given(update_weight), s = given(scale), g = given(gate),
               w = given(weight);
  const variable_list out = residual_forward(x, u, uw, s, g, w, type, eps, keep && follow);
  if (follow) {
    auto node = node_of<ResidualNode>(x, u, uw, s, g, w);
    node->call = {x.size(0), x.size(1), x.scalar_type(), type, eps, keep, u.defined()};
    // (without weight x is not needed)
    const Tensor saved[6] = {!w.defined() ? Tensor() : keep ? out[2] : x, keep ? out[3] : u,
                             uw, s, g, w};
    for (int i = 0; i < 6; ++i) node->saved[i] = SavedVariable(saved[i], false);
    torch::autograd::set_history(out[0], node);
    torch::autograd::set_history(out[1], node);
  }
  return {maybe(out[0]), maybe(out[1])};
}

Tensor gated_activation(const Tensor &x, int kind, bool keep, bool follow) {
  const variable_list out = gated_forward(x, kind, keep && follow);
  if (follow) {
    auto node = node_of<GatedNode>(x);
    node->call = {x.size(0), x.size(1) / 2, x.scalar_type(), kind, keep};
    node->saved[0] = SavedVariable(keep ? out[1] : x, false);
    torch::autograd::set_history(out[0], node);
  }
  return out[0];
}

Tensor checkpoint_linear(const Tensor &x, const Tensor &weight, const Maybe &bias, bool direct) {
  const Tensor b = given(bias);
  auto node = node_of<LinearNode>(x, weight, b);
  node->call = {x.size(0), x.size(1), x.scalar_type(), direct};
  // (the weight's gradient alone needs x)
  node->saved[0] = SavedVariable(weight.requires_grad() ? pack(x) : Tensor(), false);
  node->saved[1] = SavedVariable(weight, false);
  Tensor out;
  {
    const at::NoGradGuard none;
    out = at::linear(x, weight, bias);
  }
  torch::autograd::set_history(out, node);
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  typedef py::call_guard<py::gil_scoped_release> Free;
  m.def("errors_are", [](py::object type) { call_error = type.release().ptr(); });
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const CallError &error) {
      PyErr_SetString(call_error ? call_error : PyExc_RuntimeError, error.what());
    }
  });
  m.def("residual_norm", &residual_norm, Free());
  m.def("gated_activation", &gated_activation, Free());
  m.def("checkpoint_linear", &checkpoint_linear, Free());
  m.def("pack", &pack, Free());
  m.def("linear_int8",
        [](const Tensor &x, const Tensor &codes, int64_t row, const Tensor &scales,
           const Maybe &bias) { return linear8(x, codes, row, scales, given(bias)); },
        Free());
  m.def("residual_norm_forward",
        [](const Tensor &x, const Maybe &update, const Maybe &update_weight, const Maybe &scale,
           const Maybe &gate, const Maybe &weight, at::ScalarType type, double eps, bool keep) {
          return maybe(residual_forward(x, given(update), given(update_weight), given(scale),
                                        given(gate), given(weight), type, eps, keep));
        },
        Free());
  m.def("gated_activation_forward",
        [](const Tensor &x, int kind, bool keep) { return maybe(gated_forward(x, kind, keep)); },
        Free());
  m.def("residual_norm_backward",
        [](const Maybe &dsum, const Maybe &dnormed, const Maybe &x, const Maybe &update,
           const Maybe &update_weight, const Maybe &scale, const Maybe &gate, const Maybe &weight,
           int64_t rows, int64_t width, at::ScalarType x_type, at::ScalarType type, double eps,
           bool kept, bool has_update) {
          return maybe(residual_backward({rows, width, x_type, type, eps, kept, has_update},
                                         given(dsum), given(dnormed), given(x), given(update),
                                         given(update_weight), given(scale), given(gate),
                                         given(weight)));
        },
        Free());
  m.def("gated_activation_backward",
        [](const Tensor &dout, const Tensor &x, int64_t rows, int64_t width, at::ScalarType type,
           int kind, bool kept) {
          return maybe(gated_backward({rows, width, type, kind, kept}, dout, x));
        },
        Free());
  m.def("checkpoint_linear_backward",
        [](const Tensor &dy, const Maybe &kept, const Tensor &weight, int64_t rows, int64_t width,
           at::ScalarType type, bool direct, bool need_x, bool need_weight, bool need_bias) {
          return maybe(linear_backward({rows, width, type, direct}, dy, given(kept), weight, need_x,
                                       need_weight, need_bias));
        },
        Free());
}
