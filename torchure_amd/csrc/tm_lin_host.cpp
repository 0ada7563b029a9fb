// tm_lin_host.cpp -- host side of the linear layers and the 8-bit activations (CPU code only).
//
// A layer's forward or backward pass is two to seven kernels with a buffer for each result. Driven from Python
// (a foreign-function call and one or two allocations for every kernel) the host took 150-300 us for a
// training pass of a small layer whose GPU work takes 60; one call into this file for each pass takes
// its place. It holds no state between calls but the entry points' addresses; every kernel is
// reached through the C ABI (include/torchure_amd.h), and arguments come checked from linear.py.

#include <torch/extension.h>
#include <torch/csrc/Exceptions.h>

#include <cstdint>
#include <string>
#include <tuple>

#include "tm_rows.h"
#include "torchure_amd.h"

namespace py = pybind11;

namespace {

using namespace tm_rows;

struct Abi {
  decltype(&tm_lin_workspace_bytes) lin_bytes;
  decltype(&tm_lin) lin;
  decltype(&tm_quantize_e4m3) quantize;
  decltype(&tm_dequantize_e4m3) dequantize;
  decltype(&tm_held_gate) held_gate;
  decltype(&tm_act_grad_workspace_bytes) act_bytes;
  decltype(&tm_act_grad) act_grad;
  decltype(&tm_last_error) last_error;
  py::object native_error;
};
Abi* g_abi = nullptr;  // set once, at the first call, under the GIL

void lin_bind(const py::dict& addresses, const py::object& native_error) {
  if (g_abi) return;
  auto at = [&](const char* name) { return reinterpret_cast<void*>(addresses[name].cast<uintptr_t>()); };
  Abi* a = new Abi();
  a->lin_bytes = reinterpret_cast<decltype(a->lin_bytes)>(at("tm_lin_workspace_bytes"));
  a->lin = reinterpret_cast<decltype(a->lin)>(at("tm_lin"));
  a->quantize = reinterpret_cast<decltype(a->quantize)>(at("tm_quantize_e4m3"));
  a->dequantize = reinterpret_cast<decltype(a->dequantize)>(at("tm_dequantize_e4m3"));
  a->held_gate = reinterpret_cast<decltype(a->held_gate)>(at("tm_held_gate"));
  a->act_bytes = reinterpret_cast<decltype(a->act_bytes)>(at("tm_act_grad_workspace_bytes"));
  a->act_grad = reinterpret_cast<decltype(a->act_grad)>(at("tm_act_grad"));
  a->last_error = reinterpret_cast<decltype(a->last_error)>(at("tm_last_error"));
  a->native_error = native_error;
  g_abi = a;
}

const Abi& abi() {
  if (!g_abi) throw std::runtime_error("torchure_amd._tm_host: lin_bind was not called");
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

bool fits(const Rows& r) {  // whole 16-byte groups, as the kernels read operands
  return r.t.scalar_type() == at::kBFloat16 && r.d % 8 == 0 && r.ld % 8 == 0 &&
         (reinterpret_cast<uintptr_t>(r.t.data_ptr()) & 15) == 0;
}

// What is kept of a matrix for the backward pass.
struct Held {
  Tensor values, exps;
};

// What the backward pass is given of it. (A saved tensor may come back in other strides than it was kept in: moved to
// the host and back, say.)
Held held_of(const Opt& values, const Opt& exps) {
  return {values ? values->contiguous() : Tensor(), exps ? exps->contiguous() : Tensor()};
}

// A weight's kept operand, whole rows of it.
Rows weight_of(const Tensor& kept, i64 rows, i64 cols) {
  const Tensor t = kept.stride(1) == 1 ? kept : kept.contiguous();
  return {t, rows, cols, rows > 1 ? t.stride(0) : t.size(1)};
}

Held room_for(int kind, i64 rows, i64 cols, const Tensor& like) {
  if (kind == TM_HELD_BF16) return {room(like, {rows, up(cols, 8)}, at::kBFloat16), {}};
  return {room(like, {rows, up(cols, 32)}, at::kByte), room(like, {(rows + 31) / 32, (cols + 31) / 32}, at::kByte)};
}

struct Call {
  const Abi& a;
  void* stream;

  // dz = dy act'(z), or dy cast, into padded bf16 rows; db its column sums. Either may be undefined.
  void act_grad(const Tensor& dz, const Tensor& db, const Rows& dy, int kind, const Held& z, int act) const {
    const size_t need = db.defined() ? a.act_bytes(dy.n, dy.d) : 0;
    Tensor ws;
    if (need) ws = room(dy.t, {static_cast<i64>(need)}, at::kByte);
    check(a.act_grad(bf16_of(dz), dz.defined() ? dz.size(1) : 0, ptr(db), db.defined() && is_f32(db), ptr(dy.t),
                     is_f32(dy.t), dy.ld, ptr(z.values), bytes_of(z.exps), z.values.defined() ? z.values.size(1) : 0, kind,
                     act, dy.n, dy.d, ptr(ws), need, stream),
          "tm_act_grad");
  }

  // A product's operand: the rows as they lie where the kernels read them so, else their bf16 values in rows
  // padded with zeros.
  Rows operand(const Rows& r) const {
    if (fits(r)) return r;
    const Tensor p = room(r.t, {r.n, up(r.d, 8)}, at::kBFloat16);
    act_grad(p, {}, r, TM_HELD_NOT, {}, TM_ACT_NONE);
    return {p, r.n, r.d, p.size(1)};
  }

  // next: 0, or TM_READ_NEXT where x is read again by what follows.
  Held quantize(const Rows& x, const Tensor& copy, int next) const {
    const Held h = room_for(TM_HELD_E4M3, x.n, x.d, x.t);
    check(a.quantize(bytes_of(h.values), bytes_of(h.exps), h.values.size(1), ptr(x.t), is_f32(x.t) | next, x.ld, x.n, x.d,
                     bf16_of(copy), copy.defined() ? copy.size(1) : 0, stream),
          "tm_quantize_e4m3");
    return h;
  }

  void dequantize(const Tensor& out, i64 ld, const Held& h, i64 rows, i64 cols, int next) const {
    check(a.dequantize(ptr(out), is_f32(out) | next, ld, bytes_of(h.values), bytes_of(h.exps), h.values.size(1), rows, cols,
                       stream),
          "tm_dequantize_e4m3");
  }

  // silu(g) u of what is held, as an operand.
  Rows held_gate(const Held& g, const Held& u, int kind, i64 cols) const {
    const i64 n = g.values.size(0), ld = up(cols, 8);
    const Tensor h = room(g.values, {n, ld}, at::kBFloat16);
    check(a.held_gate(bf16_of(h), ld, ptr(g.values), ptr(u.values), bytes_of(g.exps), bytes_of(u.exps), g.values.size(1),
                      kind, n, cols, stream),
          "tm_held_gate");
    return {h, n, cols, ld};
  }

  // The first product's operand, and what is kept of it for the weight's gradient.
  Rows input(const Rows& x, int kind, bool keep, Held* kept) const {
    if (!keep || kind == TM_HELD_BF16) {
      const Rows o = operand(x);
      if (keep) kept->values = o.t;
      return o;
    }
    if (fits(x)) {
      *kept = quantize(x, {}, TM_READ_NEXT);
      return x;
    }
    const Tensor copy = room(x.t, {x.n, up(x.d, 8)}, at::kBFloat16);
    *kept = quantize(x, copy, 0);
    return {copy, x.n, x.d, copy.size(1)};
  }

  // The bf16 operand of a kept input of `cols` columns.
  Rows kept_operand(const Tensor& values, const Opt& exps, i64 cols) const {
    const i64 n = values.size(0);
    if (!exps) return weight_of(values, n, cols);
    const Held h = held_of(values, exps);
    const i64 ld = up(cols, 8);
    Tensor p = room(h.values, {n, ld}, at::kBFloat16);
    if (ld != cols) p.narrow(1, cols, ld - cols).zero_();
    dequantize(p, ld, h, n, cols, TM_READ_NEXT);
    return {p, n, cols, ld};
  }

  void product(tm_lin_t& d, const Rows& p, const Rows& b, const Tensor& out, bool two = false) const {
    d.a = bf16_of(p.t);
    d.lda = p.ld;
    d.b0 = bf16_of(b.t);
    d.ldb = b.ld;
    d.o0 = ptr(out);
    d.ldo = out.size(1);
    d.out_f32 = is_f32(out);
    const size_t need = a.lin_bytes(d.op, d.rows, d.inp, d.out, two);
    Tensor ws;
    if (need) ws = room(out, {static_cast<i64>(need)}, at::kByte);
    check(a.lin(&d, ptr(ws), need, stream), "tm_lin");
  }
};

tm_lin_t desc(int op, i64 rows, i64 inp, i64 out) {
  tm_lin_t d = {};
  d.op = op;
  d.rows = rows;
  d.inp = inp;
  d.out = out;
  return d;
}

void hold(tm_lin_t& d, int kind, const Held& z, const Held& z1) {
  d.held = kind;
  d.z0 = ptr(z.values);
  d.s0 = bytes_of(z.exps);
  d.z1 = ptr(z1.values);
  d.s1 = bytes_of(z1.exps);
  d.ldz = z.values.size(1);
}

void set_residual(tm_lin_t& d, const Rows& r) {
  if (!r.t.defined()) return;
  d.res = ptr(r.t);
  d.ldr = r.ld;
  d.res_f32 = is_f32(r.t);
}

// A call's result in x's leading dimensions, and the same memory as rows. (The result is no view, else torch would
// refuse to change it in place.)
struct Result {
  Tensor y, rows;
};

Result result_for(const Tensor& x, i64 n, i64 out, const Rows& res) {
  std::vector<i64> s(x.sizes().begin(), x.sizes().end());
  s.back() = out;
  const Tensor y = room(x, s, res.t.defined() ? res.t.scalar_type() : at::kBFloat16);
  return {y, x.dim() == 2 ? y : y.view({n, out})};
}

// y = act(x w^T + bias) + residual. Returns (y, input kept, its exponents, z kept, its exponents, the weight's
// operand): what keep_x, keep_z and keep_w ask for.
py::tuple lin_forward(const Tensor& x, const Tensor& weight, const Opt& bias, const Opt& residual, int act, int kind,
                      bool keep_x, bool keep_z, bool keep_w, uintptr_t stream) {
  HANDLE_TH_ERRORS
  Held kept, z;
  Tensor y, w;
  without_gil([&] {
    const Call c{abi(), reinterpret_cast<void*>(stream)};
    const Rows xr = rows_of(x), wr = c.operand(rows_of(weight));
    Rows res;
    if (residual) res = rows_of(*residual);
    const Tensor b = bias ? bias->detach().resolve_neg().contiguous() : Tensor();
    const i64 out = weight.size(0);
    const Rows o = c.input(xr, kind, keep_x, &kept);
    const Result result = result_for(x, xr.n, out, res);
    y = result.y;
    tm_lin_t d = desc(TM_LIN_FORWARD, xr.n, xr.d, out);
    d.act = act;
    d.bias = ptr(b);
    d.bias_f32 = b.defined() && is_f32(b);
    set_residual(d, res);
    if (keep_z) {
      z = room_for(kind, xr.n, out, x);
      hold(d, kind, z, {});
    }
    c.product(d, o, wr, result.rows);
    if (keep_w) w = wr.t;
  });
  return py::make_tuple(y, or_none(kept.values), or_none(kept.exps), or_none(z.values), or_none(z.exps), or_none(w));
  END_HANDLE_TH_ERRORS_PYBIND
}

at::ScalarType type_of(bool f32) { return f32 ? at::kFloat : at::kBFloat16; }

// (dx, dw, db), each as asked for. x_sizes and the types are the inputs' own.
py::tuple lin_backward(const Tensor& dy, const Opt& xv, const Opt& xs, const Opt& zv, const Opt& zs, const Opt& w,
                       std::vector<i64> x_sizes, bool x_f32, bool w_f32, bool b_f32, int act, int kind, bool need_x,
                       bool need_w, bool need_b, uintptr_t stream) {
  HANDLE_TH_ERRORS
  Tensor dx, dw, db;
  without_gil([&] {
    const Call c{abi(), reinterpret_cast<void*>(stream)};
    const Rows d = rows_of(dy);
    const i64 inp = x_sizes.back();
    if (need_b) db = room(dy, {d.d}, type_of(b_f32));
    const bool products = need_x || need_w;
    Rows dz = d;
    if (act || (products && !fits(d))) {
      if (products) dz = {room(dy, {d.n, up(d.d, 8)}, at::kBFloat16), d.n, d.d, up(d.d, 8)};
      c.act_grad(products ? dz.t : Tensor(), db, d, act ? kind : TM_HELD_NOT, act ? held_of(zv, zs) : Held{}, act);
    } else if (need_b) {
      c.act_grad({}, db, d, TM_HELD_NOT, {}, TM_ACT_NONE);
    }
    if (need_x) {
      dx = room(dy, {d.n, inp}, type_of(x_f32));
      tm_lin_t p = desc(TM_LIN_GRAD_X, d.n, inp, d.d);
      c.product(p, dz, weight_of(*w, d.d, inp), dx);
      dx = dx.view(x_sizes);
    }
    if (need_w) {
      dw = room(dy, {d.d, inp}, type_of(w_f32));
      tm_lin_t p = desc(TM_LIN_GRAD_W, d.n, inp, d.d);
      c.product(p, dz, c.kept_operand(*xv, xs, inp), dw);
    }
  });
  return py::make_tuple(or_none(dx), or_none(dw), or_none(db));
  END_HANDLE_TH_ERRORS_PYBIND
}

// The gate's and up's weights with equal row strides, which a product of both reads them in. (Operands of different
// strides are rows of d, a multiple of 8, or d's next one.)
std::pair<Rows, Rows> alike(Rows g, Rows u) {
  if (g.ld != u.ld) {  // one strided, one not: both into rows of their own
    const i64 wide = up(g.d, 8);
    g = {g.t.narrow(1, 0, wide).contiguous(), g.n, g.d, wide};
    u = {u.t.narrow(1, 0, wide).contiguous(), u.n, u.d, wide};
  }
  return {g, u};
}

// Returns (y, input kept, its exponents, gate kept, exponents, up kept, exponents, the three weights' operands).
py::tuple mlp_forward(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down,
                      const Opt& residual, int kind, bool keep_x, bool keep_z, bool keep_in, bool keep_down,
                      uintptr_t stream) {
  HANDLE_TH_ERRORS
  Held kept, g, u;
  Tensor y, wg, wu, wd;
  without_gil([&] {
    const Call c{abi(), reinterpret_cast<void*>(stream)};
    const Rows xr = rows_of(x), dr = c.operand(rows_of(w_down));
    const auto in = alike(c.operand(rows_of(w_gate)), c.operand(rows_of(w_up)));
    Rows res;
    if (residual) res = rows_of(*residual);
    const i64 ffn = w_gate.size(0), out = w_down.size(0);
    const Rows o = c.input(xr, kind, keep_x, &kept);
    tm_lin_t d = desc(TM_LIN_GATE, xr.n, xr.d, ffn);
    d.b1 = bf16_of(in.second.t);
    if (keep_z) {
      g = room_for(kind, xr.n, ffn, x);
      u = room_for(kind, xr.n, ffn, x);
      hold(d, kind, g, u);
    }
    const Rows h = {room(x, {xr.n, up(ffn, 8)}, at::kBFloat16), xr.n, ffn, up(ffn, 8)};
    c.product(d, o, in.first, h.t);
    const Result result = result_for(x, xr.n, out, res);
    y = result.y;
    tm_lin_t e = desc(TM_LIN_FORWARD, xr.n, ffn, out);
    set_residual(e, res);
    c.product(e, h, dr, result.rows);
    if (keep_in) {
      wg = in.first.t;
      wu = in.second.t;
    }
    if (keep_down) wd = dr.t;
  });
  return py::make_tuple(y, or_none(kept.values), or_none(kept.exps), or_none(g.values), or_none(g.exps),
                        or_none(u.values), or_none(u.exps), or_none(wg), or_none(wu), or_none(wd));
  END_HANDLE_TH_ERRORS_PYBIND
}

// (dx, dw_gate, dw_up, dw_down), each as asked for.
py::tuple mlp_backward(const Tensor& dy, const Opt& xv, const Opt& xs, const Tensor& gv, const Opt& gs, const Tensor& uv,
                       const Opt& us, const Opt& wg, const Opt& wu, const Opt& wd, std::vector<i64> x_sizes, i64 ffn,
                       bool x_f32, bool g_f32, bool u_f32, bool d_f32, int kind, bool need_x, bool need_g, bool need_u,
                       bool need_d, uintptr_t stream) {
  HANDLE_TH_ERRORS
  Tensor dx, dg, du, dd;
  without_gil([&] {
    const Call c{abi(), reinterpret_cast<void*>(stream)};
    const Rows a = c.operand(rows_of(dy));
    const i64 n = a.n, out = a.d, dim = x_sizes.back(), pad = up(ffn, 64);
    const Held g = held_of(gv, gs), u = held_of(uv, us);
    // [d_gate | d_up], where a gradient behind them is wanted, and the down projection's input again
    Rows both = {Tensor(), n, ffn, 2 * pad}, h = {Tensor(), n, ffn, pad};
    if (need_x || need_g || need_u) {
      both.t = room(dy, {n, 2 * pad}, at::kBFloat16);
      if (need_d) h.t = room(dy, {n, pad}, at::kBFloat16);
      tm_lin_t p = desc(TM_LIN_GATE_GRAD, n, ffn, out);
      hold(p, kind, g, u);
      p.o1 = ptr(h.t);
      p.ldo1 = pad;
      c.product(p, a, weight_of(*wd, out, ffn), both.t);
    } else if (need_d) {
      h = c.held_gate(g, u, kind, ffn);
    }
    if (need_d) {
      dd = room(dy, {out, ffn}, type_of(d_f32));
      tm_lin_t q = desc(TM_LIN_GRAD_W, n, ffn, out);
      c.product(q, a, h, dd);
      h.t = Tensor();
    }
    if (need_x) {
      dx = room(dy, {n, dim}, type_of(x_f32));
      tm_lin_t q = desc(TM_LIN_GRAD_X, n, dim, ffn);
      const auto in = alike(weight_of(*wg, ffn, dim), weight_of(*wu, ffn, dim));
      q.b1 = bf16_of(in.second.t);
      c.product(q, both, in.first, dx, true);
      dx = dx.view(x_sizes);
    }
    if (need_g || need_u) {
      const Rows xb = c.kept_operand(*xv, xs, dim);
      if (need_g) dg = room(dy, {ffn, dim}, type_of(g_f32));
      if (need_u) du = room(dy, {ffn, dim}, type_of(u_f32));
      if (need_g && need_u && g_f32 == u_f32) {
        tm_lin_t q = desc(TM_LIN_GRAD_W, n, dim, ffn);
        q.o1 = ptr(du);
        q.ldo1 = dim;
        c.product(q, both, xb, dg, true);
      } else {
        for (int i = 0; i < 2; ++i) {
          const Tensor& dst = i ? du : dg;
          if (!dst.defined()) continue;
          tm_lin_t q = desc(TM_LIN_GRAD_W, n, dim, ffn);
          c.product(q, {both.t.narrow(1, i * pad, pad), n, ffn, 2 * pad}, xb, dst);
        }
      }
    }
  });
  return py::make_tuple(or_none(dx), or_none(dg), or_none(du), or_none(dd));
  END_HANDLE_TH_ERRORS_PYBIND
}

// (values, exponents) of a tensor with elements.
py::tuple act_quantize(const Tensor& x, uintptr_t stream) {
  HANDLE_TH_ERRORS
  Held h;
  without_gil([&] {
    const Call c{abi(), reinterpret_cast<void*>(stream)};
    h = c.quantize(rows_of(x), {}, 0);
  });
  return py::make_tuple(h.values, h.exps);
  END_HANDLE_TH_ERRORS_PYBIND
}

Tensor act_dequantize(const Tensor& values, const Tensor& exps, std::vector<i64> sizes, bool f32, uintptr_t stream) {
  HANDLE_TH_ERRORS
  Tensor out;
  without_gil([&] {
    const Call c{abi(), reinterpret_cast<void*>(stream)};
    out = room(values, sizes, type_of(f32));
    const i64 cols = sizes.back();
    if (out.numel()) c.dequantize(out, cols, {values, exps}, out.numel() / cols, cols, 0);
  });
  return out;
  END_HANDLE_TH_ERRORS_PYBIND
}

// Whether the tensors that are given are plain, on the current device and bf16 or fp32 where that may be:
// a call with these and matching shapes needs none of linear.py's other checks.
bool lin_plain(const Tensor& x, const std::vector<Tensor>& weights, const Opt& bias, const Opt& residual, i64 out,
               int current_device) {
  auto good = [&](const Tensor& t) { return t.is_cuda() && t.device().index() == current_device; };
  if (!good(x) || x.scalar_type() != at::kBFloat16 || x.dim() < 1 || x.numel() == 0) return false;
  for (const Tensor& w : weights)
    if (!good(w) || w.scalar_type() != at::kBFloat16 || w.dim() != 2 || w.numel() == 0) return false;
  if (bias) {
    if (!good(*bias) || bias->dim() != 1 || bias->size(0) != out ||
        (bias->scalar_type() != at::kBFloat16 && !is_f32(*bias)))
      return false;
  }
  if (residual) {
    if (!good(*residual) || residual->dim() != x.dim() || residual->size(-1) != out ||
        (residual->scalar_type() != at::kBFloat16 && !is_f32(*residual)))
      return false;
    for (i64 i = 0; i + 1 < x.dim(); ++i)
      if (residual->size(i) != x.size(i)) return false;
  }
  return true;
}

}  // namespace

void tm_lin_host_bind(py::module_& m) {
  m.def("lin_bind", &lin_bind, "addresses of the C ABI's linear-layer entry points, and the exception of a failed call");
  m.def("lin_forward", &lin_forward, "the forward pass of a linear layer");
  m.def("lin_backward", &lin_backward, "its gradients");
  m.def("mlp_forward", &mlp_forward, "the forward pass of the gated feed-forward");
  m.def("mlp_backward", &mlp_backward, "its gradients");
  m.def("act_quantize", &act_quantize, "a tensor in 8 bits");
  m.def("act_dequantize", &act_dequantize, "and back");
  m.def("lin_plain", &lin_plain, "whether a call needs none of the other checks");
}
