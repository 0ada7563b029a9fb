// tm_rows.h -- what the host sides of the operators share: tensors as rows, new tensors, failed entry points.
#ifndef TM_ROWS_H
#define TM_ROWS_H

#include <torch/extension.h>

#include <cstdint>
#include <stdexcept>
#include <string>

namespace tm_rows {

namespace py = pybind11;
using i64 = int64_t;
using at::Tensor;
using Opt = c10::optional<Tensor>;

// A C entry point's status was not TM_OK; becomes torchure_amd._native.NativeError.
struct EntryFailed : std::runtime_error {
  using std::runtime_error::runtime_error;
};

inline i64 up(i64 n, i64 to) { return (n + to - 1) / to * to; }
inline bool is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
inline char* ptr(const Tensor& t) { return t.defined() ? static_cast<char*>(t.data_ptr()) : nullptr; }
inline uint8_t* bytes_of(const Tensor& t) { return reinterpret_cast<uint8_t*>(ptr(t)); }
inline uint16_t* bf16_of(const Tensor& t) { return reinterpret_cast<uint16_t*>(ptr(t)); }
inline py::object or_none(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

inline Tensor room(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type).requires_grad(false).memory_format(c10::nullopt));
}

// A tensor as rows of its last dimension, the elements of a row next to each other, rows apart by at least their
// length and less than 2^23 elements. (The tensor is kept alive by its own storage where no copy is made.)
struct Rows {
  Tensor t;
  i64 n = 0, d = 0, ld = 0;
};

inline Rows rows_of(const Tensor& given) {
  Tensor t = given.detach();
  if (t.is_neg()) t = t.resolve_neg();
  const i64 d = t.size(-1), n = d ? t.numel() / d : 0;
  if (t.dim() != 2) t = t.reshape({n, d});
  if ((d > 1 && t.stride(1) != 1) || (n > 1 && (t.stride(0) < d || t.stride(0) >= (1 << 23))))
    t = t.contiguous();
  return {t, n, d, n > 1 ? t.stride(0) : d};
}

}  // namespace tm_rows

#endif
