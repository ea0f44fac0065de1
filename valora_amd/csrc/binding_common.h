// What the torch binding's sources share: errors, operand types, calls without the interpreter lock.
#pragma once

#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "mlora.h"

namespace py = pybind11;

[[noreturn]] inline void raise(const std::string &msg) { throw std::runtime_error(msg); }

inline void check_rc(int rc) {
  if (rc == MLORA_OK) return;
  const char *m = mlora_last_error();
  raise((m && *m) ? std::string(m) : "libmlora call failed with status " + std::to_string(rc));
}

inline mlora_dtype dtype_code(const at::Tensor &t) {
  if (t.scalar_type() == at::kHalf) return MLORA_F16;
  if (t.scalar_type() == at::kBFloat16) return MLORA_BF16;
  return (mlora_dtype)-1;
}

inline std::string dtype_name(const at::Tensor &t) { return std::string("torch.") + c10::toString(t.scalar_type()); }

// A C call without the interpreter lock (a launch waits where the device's queue is full, and other Python threads go on
// meanwhile).
template <typename F>
void check_unlocked(F call) {
  int rc;
  {
    py::gil_scoped_release unlocked;
    rc = call();
  }
  check_rc(rc);   // (the message belongs to this thread)
}

void bind_attention(py::module_ &m);   // binding_attention.cpp
