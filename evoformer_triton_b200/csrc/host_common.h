// What the native boundaries share (host.cpp: the attention; host_inputs.cpp: the operators before it; host_sequences.cpp:
// packed sequences).
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <stdexcept>
#include <string>
#include <vector>

#include "evoattn.h"

namespace evohost {

using at::Tensor;
using Maybe = c10::optional<Tensor>;

inline void check(int rc, const char* what) {
  if (rc != EVOATTN_OK) throw std::runtime_error(std::string(what) + " failed: " + evoattn_strerror(rc) + " (status " + std::to_string(rc) + ")");
}
inline int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? EVOATTN_BF16 : t == at::kHalf ? EVOATTN_FP16 : EVOATTN_FP32; }
inline bool known(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

[[noreturn]] inline void raise(PyObject* type, const char* text) {
  PyErr_SetString(type, text);
  throw py::error_already_set();
}

[[noreturn]] inline void type_error(const std::string& text) { raise(PyExc_TypeError, text.c_str()); }
[[noreturn]] inline void value_error(const std::string& text) { raise(PyExc_ValueError, text.c_str()); }
[[noreturn]] inline void runtime_error(const std::string& text) { raise(PyExc_RuntimeError, text.c_str()); }

inline void check_main(const Tensor& t, const char* op, const char* name) {
  // A tracer would record the allocation of the result, not the call.
  if (torch::jit::tracer::isTracing()) runtime_error(std::string(op) + " cannot be traced");
  if (!t.is_cuda()) runtime_error(std::string(op) + " runs on CUDA tensors only; there is no CPU fallback");
  if (!known(t.scalar_type())) type_error(std::string(name) + " must be bfloat16, float16 or float32");
}
// A small dense tensor of weights beside t, of any of the three types.
inline void check_weight(const Tensor& w, const Tensor& t, const char* name, at::IntArrayRef shape) {
  if (w.device() != t.device()) runtime_error(std::string(name) + " is on " + w.device().str() + ", not on " + t.device().str());
  if (!known(w.scalar_type())) type_error(std::string(name) + " must be bfloat16, float16 or float32");
  if (w.sizes() != shape) {
    std::string s = std::string(name) + " must have the shape [";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    value_error(s + "]");
  }
}
// Sizes are 32-bit in the C ABI: a view of many times the same values may have more along an axis.
inline void check_sizes(at::IntArrayRef sizes, int64_t most, const char* text) {
  for (const int64_t n : sizes)
    if (n > most) value_error(text);
}
inline float checked_eps(double eps) {
  if (!(eps >= 0.0) || std::isinf(eps)) value_error("eps must be a finite number that is not negative");
  return (float)eps;
}
// Derivatives in forward mode (dual tensors) are not worked out.  A dual tensor need not require a gradient, so a call that
// took it as an ordinary one would return a result whose derivative is zero; the same goes for a dual gradient.
inline bool is_dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
inline std::string no_forward_mode(const char* op) { return std::string(op) + " has no derivative in forward mode"; }
inline void no_duals(const char* op, std::initializer_list<const Maybe*> inputs) {
  for (const Maybe* t : inputs)
    if (*t && is_dual(**t)) runtime_error(no_forward_mode(op));
}
inline void once(const char* op, const Tensor& grad) {
  if (is_dual(grad)) throw std::runtime_error(no_forward_mode(op));
  if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(op) + " can be differentiated once; its gradient has no graph (create_graph)");
}
inline bool wants_grad(std::initializer_list<const Maybe*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Maybe* t : inputs)
    if (*t && (*t)->requires_grad()) return true;
  return false;
}
inline const void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// Memory holds the values of a tensor but where it is a view that has yet to be negated, as the imaginary part of a conjugate is.
inline Tensor dense(const Maybe& t) { return t ? t->resolve_neg().contiguous() : Tensor(); }
inline Tensor last_axis_dense(const Tensor& t) {
  const Tensor r = t.resolve_neg();
  return r.dim() == 0 || r.size(-1) <= 1 || r.stride(-1) == 1 ? r : r.contiguous();
}

// The axes before the last one as three (or fewer) with strides; false where that takes more.
inline bool three_axes(const Tensor& t, int64_t* n, int64_t* st) {
  int used = 0;
  int64_t size[3] = {1, 1, 1}, stride[3] = {0, 0, 0};  // innermost first
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (used && t.stride(d) == stride[used - 1] * size[used - 1]) {
      size[used - 1] *= t.size(d);
      continue;
    }
    if (used == 3) return false;
    size[used] = t.size(d);
    stride[used++] = t.stride(d);
  }
  for (int i = 0; i < 3; ++i) n[2 - i] = size[i], st[2 - i] = stride[i];
  return true;
}
inline Tensor rows_in_place(const Tensor& t, int64_t* n, int64_t* st) {
  Tensor r = last_axis_dense(t);
  if (three_axes(r, n, st)) return r;
  r = r.contiguous();
  three_axes(r, n, st);
  return r;
}

// (host.cpp) The word of a device that kernels set when they give up a bounded wait; whether every call goes to the
// CUDA-core kernels; and what the last call of either direction reported.
int32_t* status_ptr(c10::Device dev);
bool generic_forced();
void note_call(bool bwd);

void register_inputs(py::module& m);
void register_sequences(py::module& m);

}  // namespace evohost
