// tm_layer_host.cpp -- host side of the norms and the embedding (CPU code only): makes the results and workspaces and reaches the kernels
// through the C ABI (include/torchure_amd.h). The autograd functions are C++ too: a norm's kernels take 10 to 100 us, and a
// function in Python, with the lock that its backward pass takes on the engine's thread, as much again on the host. Arguments come checked
// from norm.py and embed.py.

#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
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
  decltype(&tm_embed_lookup) lookup;
  decltype(&tm_embed_grad_workspace_bytes) embed_bytes;
  decltype(&tm_embed_grad) embed_grad;
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
  a->lookup = reinterpret_cast<decltype(a->lookup)>(at("tm_embed_lookup"));
  a->embed_bytes = reinterpret_cast<decltype(a->embed_bytes)>(at("tm_embed_grad_workspace_bytes"));
  a->embed_grad = reinterpret_cast<decltype(a->embed_grad)>(at("tm_embed_grad"));
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

// The stream that a backward pass runs on: the engine makes the forward pass's the current one, and a node that is called
// directly runs where its caller is.
void* current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

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

struct NormFunction : torch::autograd::Function<NormFunction> {
  enum : i64 { kLayer = 1, kWeight = 2, kWeightF32 = 4, kBias = 8, kBiasF32 = 16, kXF32 = 32 };

  // Kept are, for x's gradient, x, the statistics and the weight; for the weight's, x and the statistics; for the bias's nothing.
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& weight, const Opt& bias, const Norm& n) {
    const bool for_x = wants_grad(x), for_weight = weight && wants_grad(*weight);
    variable_list kept(3);
    const Tensor y = norm_forward(x, weight, bias, n, for_x || for_weight ? &kept : nullptr);
    if (!for_x) kept[2] = Tensor();
    ctx->save_for_backward(std::move(kept));
    ctx->saved_data["flags"] = (n.layer ? kLayer : 0) | (is_f32(x) ? kXF32 : 0) | (weight ? kWeight | (is_f32(*weight) ? kWeightF32 : 0) : 0) |
                               (bias ? kBias | (is_f32(*bias) ? kBiasF32 : 0) : 0);
    return y;
  }

  // (A saved tensor may come back in other strides than it was kept in.)
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& dy = grads[0];
    const variable_list kept = ctx->get_saved_variables();
    const i64 flags = ctx->saved_data["flags"].toInt();
    const bool layer = flags & kLayer, has_w = flags & kWeight, has_b = flags & kBias, x_f32 = flags & kXF32;
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1),
               need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    Tensor dx, dw, db;
    {
      const at::AutoGradMode no_grad(false);
      const OnDevice on(dy);
      const Rows d = rows_of(dy), r = kept[0].defined() ? rows_of(kept[0]) : Rows{Tensor(), d.n, d.d, d.d};
      const Tensor s = kept[1].defined() ? kept[1].contiguous() : Tensor(), w = kept[2].defined() ? kept[2].contiguous() : Tensor();
      if (need_x) dx = room(dy, dy.sizes(), type_of(x_f32));
      if (need_w) dw = room(dy, {d.d}, type_of(flags & kWeightF32));
      if (need_b) db = room(dy, {d.d}, type_of(flags & kBiasF32));
      const size_t need = need_w || need_b ? abi().norm_bytes(d.n, d.d, x_f32, is_f32(d.t), layer) : 0;
      Tensor ws;
      if (need) ws = room(dy, {static_cast<i64>(need)}, at::kByte);
      const float* rstd = s.defined() ? s.data_ptr<float>() : nullptr;
      check(abi().norm_backward(ptr(dx), ptr(dw), ptr(db), f32_if(db), ptr(d.t), is_f32(d.t), d.ld, ptr(r.t), x_f32, r.ld, rstd,
                                layer && rstd ? rstd + d.n : nullptr, ptr(w), f32_if(w), f32_if(dw), layer, d.n, d.d, ptr(ws), need,
                                current_stream(dy)),
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

// ---------------------------------------------------------------- embedding

struct Embed {
  double scale;
  i64 padding;
  bool y_f32;
  void* stream;
};

bool wide(const Tensor& ids) { return ids.scalar_type() == at::kLong; }

Tensor lookup(const Tensor& ids, const Tensor& weight, const Embed& e) {
  const OnDevice on(weight);
  const Rows w = rows_of(weight);
  std::vector<i64> sizes(ids.sizes().begin(), ids.sizes().end());
  sizes.push_back(w.d);
  const Tensor y = room(weight, sizes, type_of(e.y_f32));
  check(abi().lookup(ptr(y), e.y_f32, ptr(w.t), is_f32(w.t), w.ld, ptr(ids), wide(ids), ids.numel(), w.n, w.d,
                     static_cast<float>(e.scale), e.stream),
        "tm_embed_lookup");
  return y;
}

// dw = the gradient, or, with `add`, dw += it.
void table_grad(const Tensor& dw, i64 ldw, const Tensor& dy, const Tensor& ids, double scale, i64 padding, bool add, void* stream) {
  const OnDevice on(dy);
  const Rows d = rows_of(dy);
  const size_t need = abi().embed_bytes(ids.numel(), dw.size(0), dw.size(1));
  const Tensor ws = room(dy, {static_cast<i64>(need)}, at::kByte);
  check(abi().embed_grad(ptr(dw), is_f32(dw), ldw, ptr(d.t), is_f32(d.t), d.ld, ptr(ids), wide(ids), ids.numel(), dw.size(0),
                         dw.size(1), static_cast<float>(scale), padding, add, ptr(ws), need, stream),
        "tm_embed_grad");
}

struct EmbedFunction : torch::autograd::Function<EmbedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, const Embed& e) {
    const Tensor kept = ids.contiguous();
    ctx->save_for_backward({kept});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["f32"] = is_f32(weight);
    ctx->saved_data["scale"] = e.scale;
    ctx->saved_data["padding"] = e.padding;
    return lookup(kept, weight, e);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& dy = grads[0];
    const Tensor ids = ctx->get_saved_variables()[0].contiguous();
    Tensor dw;
    {
      const at::AutoGradMode no_grad(false);
      dw = room(dy, {ctx->saved_data["vocab"].toInt(), dy.size(-1)}, type_of(ctx->saved_data["f32"].toBool()));
      table_grad(dw, dw.size(1), dy, ids, ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), false,
                 current_stream(dy));
    }
    return once({Tensor(), dw, Tensor()});
  }
};

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, i64 padding, bool y_f32, uintptr_t stream) {
  HANDLE_TH_ERRORS
  return without_gil([&] {
    const Embed e = {scale, padding, y_f32, reinterpret_cast<void*>(stream)};
    const bool record = at::GradMode::is_enabled() && wants_grad(weight);
    return record ? EmbedFunction::apply(ids, weight, e) : lookup(ids.contiguous(), weight, e);
  });
  END_HANDLE_TH_ERRORS_PYBIND
}

void embedding_grad(const Tensor& grad, const Tensor& ids, const Tensor& dy, double scale, i64 padding, uintptr_t stream) {
  HANDLE_TH_ERRORS
  without_gil([&] {
    const at::AutoGradMode no_grad(false);
    table_grad(grad, grad.size(0) > 1 ? grad.stride(0) : grad.size(1), dy, ids.contiguous(), scale, padding, true,
               reinterpret_cast<void*>(stream));
  });
  END_HANDLE_TH_ERRORS_PYBIND
}

// As norm_plain, for a lookup.
bool embedding_plain(const Tensor& ids, const Tensor& weight, int device) {
  return plain(weight, device) && weight.dim() == 2 && weight.numel() > 0 && ids.is_cuda() && ids.layout() == at::kStrided &&
         ids.device().index() == device && (wide(ids) || ids.scalar_type() == at::kInt) && ids.numel() > 0;
}

}  // namespace

void tm_layer_host_bind(py::module_& m) {
  m.def("layer_bind", &layer_bind, "addresses of the C ABI's norm and embedding entry points, and the exception of a failed call");
  m.def("norm", &norm, "a norm, with its gradients where they are wanted");
  m.def("embedding", &embedding, "rows of a table by id, with the table's gradient where it is wanted");
  m.def("embedding_grad", &embedding_grad, "the table's gradient, added to one that is there");
  m.def("embedding_plain", &embedding_plain, "whether a lookup needs none of the other checks");
  m.def("norm_plain", &norm_plain, "whether a call needs none of the other checks");
}
