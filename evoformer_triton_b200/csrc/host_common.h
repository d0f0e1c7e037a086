// What the native boundaries share (host.cpp: the attention; host_inputs.cpp: the operators before it).
#pragma once
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

void register_inputs(py::module& m);

}  // namespace evohost
