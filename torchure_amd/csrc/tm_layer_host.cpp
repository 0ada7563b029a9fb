// tm_layer_host.cpp -- host side of the norms (CPU code only): makes the results and workspaces and reaches the kernels
// through the C ABI (include/torchure_amd.h). The autograd functions are C++ too: a norm's kernels take 10 to 100 us, and a
// function in Python, with the lock that its backward pass takes on the engine's thread, as much again on the host. Arguments come checked
// from norm.py.

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/Exceptions.h>

#include <cstdint>
#include <string>
#include <vector>

#include "tm_rows.h"
#include "torchure_amd.h"

namespace {

using namespace tm_rows;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Abi {
  decltype(&tm_norm_forward) norm_forward;
  decltype(&tm_norm_workspace_bytes) norm_bytes;
  decltype(&tm_norm_backward) norm_backward;
  decltype(&tm_last_error) last_error;
  py::object native_error;
};
Abi* g_abi = nullptr;  // set once, at the first call, under the GIL

void layer_bind(const py::dict& addresses, const py::object& native_error) {
  if (g_abi) return;
  auto at = [&](const char* name) { return reinterpret_cast<void*>(addresses[name].cast<uintptr_t>()); };
  Abi* a = new Abi();
  a->norm_forward = reinterpret_cast<decltype(a->norm_forward)>(at("tm_norm_forward"));
  a->norm_bytes = reinterpret_cast<decltype(a->norm_bytes)>(at("tm_norm_workspace_bytes"));
  a->norm_backward = reinterpret_cast<decltype(a->norm_backward)>(at("tm_norm_backward"));
  a->last_error = reinterpret_cast<decltype(a->last_error)>(at("tm_last_error"));
  a->native_error = native_error;
  g_abi = a;
}

const Abi& abi() {
  if (!g_abi) throw std::runtime_error("torchure_amd._tm_host: layer_bind was not called");
  return *g_abi;
}

void check(int rc, const char* what) {
  if (rc != 0)
    throw EntryFailed(std::string(what) + " failed (" + std::to_string(rc) + "): " + abi().last_error());
}

// Runs body without the GIL; a failed entry point becomes torchure_amd._native.NativeError.
template <typename Body>
auto without_gil(Body&& body) -> decltype(body()) {
  try {
    py::gil_scoped_release released;
    return body();
  } catch (const EntryFailed& e) {  // the GIL is held again
    PyErr_SetString(abi().native_error.ptr(), e.what());
    throw py::error_already_set();
  }
}

at::ScalarType type_of(bool f32) { return f32 ? at::kFloat : at::kBFloat16; }
Tensor values_of(const Opt& t) { return t ? t->detach().resolve_neg().contiguous() : Tensor(); }
bool f32_if(const Tensor& t) { return t.defined() && is_f32(t); }

// A call's tensors are on one device, which its kernels are looked up on and its results made on.
struct OnDevice {
  c10::OptionalDeviceGuard guard;
  explicit OnDevice(const Tensor& t) : guard(t.device()) {}
};

// What a backward pass returned, in a pass that records itself (create_graph): a second derivative is refused, where a
// result without a graph would drop it.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once (once_differentiable)",
      static_cast<i64>(grads.size()));
  return refuse->apply(std::move(grads));
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

struct Norm {
  bool layer;
  double eps;
  bool y_f32;
  void* stream;
};

// y = norm(x) w + b in x's leading dimensions; with `kept`: x's rows, the statistics (rstd, then the means) and the
// weight.
Tensor norm_forward(const Tensor& x, const Opt& weight, const Opt& bias, const Norm& n, variable_list* kept) {
  const OnDevice on(x);
  const Rows r = rows_of(x);
  const Tensor w = values_of(weight), b = values_of(bias);
  const Tensor y = room(x, x.sizes(), type_of(n.y_f32));
  Tensor stats;
  if (kept) {
    stats = room(x, {n.layer ? 2 : 1, r.n}, at::kFloat);
    *kept = {r.t, stats, w};
  }
  float* rstd = kept ? stats.data_ptr<float>() : nullptr;
  check(abi().norm_forward(ptr(y), n.y_f32, rstd, kept && n.layer ? rstd + r.n : nullptr, ptr(r.t), is_f32(r.t), r.ld, ptr(w),
                           f32_if(w), ptr(b), f32_if(b), n.layer, n.eps, r.n, r.d, n.stream),
        "tm_norm_forward");
  return y;
}

// The engine runs a node's backward pass on the stream that its forward pass ran on, so the handle is kept.
struct NormFunction : torch::autograd::Function<NormFunction> {
  enum : i64 { kLayer = 1, kWeight = 2, kWeightF32 = 4, kBias = 8, kBiasF32 = 16 };

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& weight, const Opt& bias, const Norm& n) {
    variable_list kept;
    const Tensor y = norm_forward(x, weight, bias, n, &kept);
    ctx->save_for_backward(std::move(kept));
    ctx->saved_data["flags"] = (n.layer ? kLayer : 0) | (weight ? kWeight | (is_f32(*weight) ? kWeightF32 : 0) : 0) |
                               (bias ? kBias | (is_f32(*bias) ? kBiasF32 : 0) : 0);
    ctx->saved_data["stream"] = reinterpret_cast<i64>(n.stream);
    return y;
  }

  // (A saved tensor may come back in other strides than it was kept in.)
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& dy = grads[0];
    const variable_list kept = ctx->get_saved_variables();
    const i64 flags = ctx->saved_data["flags"].toInt();
    const bool layer = flags & kLayer, has_w = flags & kWeight, has_b = flags & kBias;
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1),
               need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    Tensor dx, dw, db;
    {
      const at::AutoGradMode no_grad(false);
      const OnDevice on(dy);
      const Rows r = rows_of(kept[0]), d = rows_of(dy);
      const Tensor s = kept[1].contiguous(), w = kept[2].defined() ? kept[2].contiguous() : Tensor();
      if (need_x) dx = room(dy, dy.sizes(), r.t.scalar_type());
      if (need_w) dw = room(dy, {r.d}, type_of(flags & kWeightF32));
      if (need_b) db = room(dy, {r.d}, type_of(flags & kBiasF32));
      const size_t need = need_w || need_b ? abi().norm_bytes(r.n, r.d, is_f32(r.t), is_f32(d.t), layer) : 0;
      Tensor ws;
      if (need) ws = room(dy, {static_cast<i64>(need)}, at::kByte);
      const float* rstd = s.data_ptr<float>();
      check(abi().norm_backward(ptr(dx), ptr(dw), ptr(db), f32_if(db), ptr(d.t), is_f32(d.t), d.ld, ptr(r.t), is_f32(r.t), r.ld,
                                rstd, layer ? rstd + r.n : nullptr, ptr(w), f32_if(w), f32_if(dw), layer, r.n, r.d, ptr(ws),
                                need, reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())),
            "tm_norm_backward");
    }
    return once({dx, dw, db, Tensor()});
  }
};

Tensor norm(const Tensor& x, const Opt& weight, const Opt& bias, bool layer, double eps, bool y_f32, uintptr_t stream) {
  HANDLE_TH_ERRORS
  return without_gil([&] {
    const Norm n = {layer, eps, y_f32, reinterpret_cast<void*>(stream)};
    const bool record = at::GradMode::is_enabled() && (wants_grad(x) || (weight && wants_grad(*weight)) || (bias && wants_grad(*bias)));
    return record ? NormFunction::apply(x, weight, bias, n) : norm_forward(x, weight, bias, n, nullptr);
  });
  END_HANDLE_TH_ERRORS_PYBIND
}

bool plain(const Tensor& t, int device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.device().index() == device &&
         (t.scalar_type() == at::kBFloat16 || is_f32(t));
}

// Whether the tensors are plain, on the current device, bf16 or fp32 and of matching shapes: such a call needs none of
// norm.py's other checks.
bool norm_plain(const Tensor& x, const Opt& weight, const Opt& bias, int device) {
  if (!plain(x, device) || x.dim() < 1 || x.numel() == 0 || x.size(-1) > 16384) return false;
  for (const Opt* p : {&weight, &bias})
    if (*p && (!plain(**p, device) || (*p)->dim() != 1 || (*p)->size(0) != x.size(-1))) return false;
  return true;
}

}  // namespace

void tm_layer_host_bind(py::module_& m) {
  m.def("layer_bind", &layer_bind, "addresses of the C ABI's norm entry points, and the exception of a failed call");
  m.def("norm", &norm, "a norm, with its gradients where they are wanted");
  m.def("norm_plain", &norm_plain, "whether a call needs none of the other checks");
}
