// Shared by the parts of the native Python entry points.
#pragma once

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/extension.h>

#include "../../include/monarch_attention_b200.h"

namespace ma_torch {

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MA_B200_F32;
    case at::kBFloat16: return MA_B200_BF16;
    case at::kHalf: return MA_B200_F16;
    default: return -1;
  }
}

inline void raise_for_status(int code) {
  if (code == MA_B200_OK) return;
  const std::string msg = std::string("monarch_attention_b200: ") + ma_b200_status_string(code) + ": " + ma_b200_last_error();
  TORCH_CHECK_VALUE(code != MA_B200_INVALID_ARGUMENT && code != MA_B200_UNSUPPORTED && code != MA_B200_WORKSPACE_TOO_SMALL, msg);
  TORCH_CHECK(false, msg);
}

inline ma_b200_tensor view4(const at::Tensor& t) {
  const auto s = t.strides();
  return {t.data_ptr(), s[0], s[1], s[2]};
}

inline at::Tensor unit_inner(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// Whether forward-mode differentiation has a tangent for t.
inline bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
inline void check_no_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), name, " has a tangent: there is no forward-mode derivative of this operator");
}

// Entry points of ma_torch_cache.cpp.
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_attend(PyObject*, PyObject* const* args, Py_ssize_t n);

}  // namespace ma_torch
