// tm_layer_host.cpp -- host side of the norms (CPU code only): as tm_lin_host.cpp does for the linear layers, one
// call into this file for each pass, which makes the results and workspaces and reaches the kernels through the C ABI
// (include/torchure_amd.h). Arguments come checked from norm.py.

#include <torch/extension.h>
#include <torch/csrc/Exceptions.h>

#include <cstdint>
#include <string>
#include <vector>

#include "tm_rows.h"
#include "torchure_amd.h"

namespace {

using namespace tm_rows;

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

// y = norm(x) w + b in x's leading dimensions. Returns (y, x's rows, statistics (rstd, then the means), the weight), the last
// three where `keep` is set, else None.
py::tuple norm_forward(const Tensor& x, const Opt& weight, const Opt& bias, bool layer, double eps, bool y_f32, bool keep,
                       uintptr_t stream) {
  HANDLE_TH_ERRORS
  Tensor y, stats, w;
  Rows r;
  without_gil([&] {
    r = rows_of(x);
    w = values_of(weight);
    const Tensor b = values_of(bias);
    y = room(x, x.sizes(), type_of(y_f32));
    if (keep) stats = room(x, {layer ? 2 : 1, r.n}, at::kFloat);
    float* rstd = keep ? stats.data_ptr<float>() : nullptr;
    check(abi().norm_forward(ptr(y), y_f32, rstd, keep && layer ? rstd + r.n : nullptr, ptr(r.t), is_f32(r.t), r.ld, ptr(w),
                             f32_if(w), ptr(b), f32_if(b), layer, eps, r.n, r.d, reinterpret_cast<void*>(stream)),
          "tm_norm_forward");
  });
  return py::make_tuple(y, keep ? or_none(r.t) : py::none(), or_none(stats), keep ? or_none(w) : py::none());
  END_HANDLE_TH_ERRORS_PYBIND
}

// (dx, dw, db), each as asked for. A saved tensor may come back in other strides than it was kept in.
py::tuple norm_backward(const Tensor& dy, const Tensor& x, const Tensor& stats, const Opt& weight, std::vector<i64> x_sizes,
                        bool layer, bool w_f32, bool b_f32, bool need_x, bool need_w, bool need_b, uintptr_t stream) {
  HANDLE_TH_ERRORS
  Tensor dx, dw, db;
  without_gil([&] {
    const Rows r = rows_of(x), d = rows_of(dy);
    const Tensor w = values_of(weight), s = stats.contiguous();
    if (need_x) dx = room(dy, x_sizes, x.scalar_type());
    if (need_w) dw = room(dy, {r.d}, type_of(w_f32));
    if (need_b) db = room(dy, {r.d}, type_of(b_f32));
    const size_t need = need_w || need_b ? abi().norm_bytes(r.n, r.d, is_f32(r.t), is_f32(d.t), layer) : 0;
    Tensor ws;
    if (need) ws = room(dy, {static_cast<i64>(need)}, at::kByte);
    const float* rstd = s.data_ptr<float>();
    check(abi().norm_backward(ptr(dx), ptr(dw), ptr(db), b_f32, ptr(d.t), is_f32(d.t), d.ld, ptr(r.t), is_f32(r.t), r.ld, rstd,
                              layer ? rstd + r.n : nullptr, ptr(w), f32_if(w), w_f32, layer, r.n, r.d, ptr(ws), need,
                              reinterpret_cast<void*>(stream)),
          "tm_norm_backward");
  });
  return py::make_tuple(or_none(dx), or_none(dw), or_none(db));
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
  m.def("norm_forward", &norm_forward, "the forward pass of a norm");
  m.def("norm_backward", &norm_backward, "its gradients");
  m.def("norm_plain", &norm_plain, "whether a call needs none of the other checks");
}
