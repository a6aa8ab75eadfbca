// What the parts of the _kv_host module that take a call's tensors as they are share: checks of layouts and types.
#pragma once

#include <c10/util/Exception.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>

namespace kv_host {

namespace py = pybind11;

constexpr int64_t kNotTaken = -2;

inline const at::Tensor* plain(const py::handle& h, int64_t device) {
  if (!THPVariable_CheckExact(h.ptr())) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(h.ptr());
  return t.is_cuda() && t.device().index() == device ? &t : nullptr;
}

inline bool index_kind(at::ScalarType t) { return t == at::kInt || t == at::kLong; }
inline bool fp8_kind(at::ScalarType t) { return t == at::kByte || t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2; }
inline bool float_kind(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
inline int float_id(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : 2; }

// The trailing [kv_heads, head_dim, block_size] of every block is packed, and no extent is empty or expanded.
inline bool packed_blocks(const at::Tensor& c) {
  const int64_t n = c.dim();
  int64_t want = 1;
  for (int64_t i = n - 1; i >= n - 3; --i) {
    if (c.size(i) < 1 || (c.size(i) != 1 && c.stride(i) != want)) return false;
    want *= c.size(i);
  }
  for (int64_t i = 0; i < n - 3; ++i)
    if (c.size(i) < 1 || (c.size(i) != 1 && c.stride(i) == 0)) return false;
  return true;
}

// Whether the bytes from one tensor's first element to its last meet another's (their elements may lie apart for all that).
inline bool spans_meet(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<uint64_t>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return reinterpret_cast<uint64_t>(a.data_ptr()) < end(b) && reinterpret_cast<uint64_t>(b.data_ptr()) < end(a);
}

// Whether a block of one of two caches of the same shape shares bytes with one of the other ([blocks, ..] or [layers,
// blocks, ..], each block packed; K and V may lie between each other in one buffer).
inline bool blocks_meet(const at::Tensor& a, const at::Tensor& b) {
  if (!spans_meet(a, b)) return false;
  const int64_t n = a.dim(), elt = a.element_size();
  const int64_t packed = a.size(n - 3) * a.size(n - 2) * a.size(n - 1) * elt;
  const int64_t apart = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
  for (int64_t i = 0; i < n - 3; ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return true;  // not looked at further
  const int64_t layers = n == 5 ? a.size(0) : 1, layer = n == 5 ? a.stride(0) * elt : 0;
  const int64_t last = a.size(n - 4) - 1, block = last > 0 ? a.stride(n - 4) * elt : 1;
  for (int64_t i = 1 - layers; i < layers; ++i) {
    const int64_t off = apart + i * layer, near = -off / block;
    for (int64_t j = near - 1; j <= near + 1; ++j) {
      const int64_t at = off + std::clamp(j, -last, last) * block;
      if (at > -packed && at < packed) return true;
    }
  }
  return false;
}

inline bool rows_packed(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

inline py::tuple not_taken() { return py::make_tuple(kNotTaken, py::none(), py::none()); }

// A call whose tensors do not fit in memory is left to Python too, which raises torch's own error for it.
template <typename... Args>
auto taken_or_left(py::tuple (*call)(Args...)) {
  return [call](Args... args) {
    try {
      return call(args...);
    } catch (const c10::OutOfMemoryError&) {
      return not_taken();
    }
  };
}

}  // namespace kv_host
