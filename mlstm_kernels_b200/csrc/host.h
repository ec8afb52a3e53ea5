// What the native host module's files share: element types, pointers and streams of tensors, errors, and the arguments of a
// Python call.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstdlib>
#include <cstring>
#include <string>

#include "calls.h"

namespace mlstm_host {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline int dtype_code(at::ScalarType t) {   // -1: not a kernel element type
  switch (t) {
    case at::kFloat: return MLSTM_F32;
    case at::kBFloat16: return MLSTM_BF16;
    case at::kHalf: return MLSTM_F16;
    default: return -1;
  }
}
inline at::ScalarType code_dtype(int code) {
  return code == MLSTM_F32 ? at::kFloat : code == MLSTM_BF16 ? at::kBFloat16 : at::kHalf;
}

inline const char* const kNeedsCuda = "mlstm_kernels_b200 kernels run on CUDA tensors only (there is no CPU fallback)";

inline Tensor empty(at::IntArrayRef size, at::ScalarType dt, const at::Device& dev) {
  return Tensor(at::detail::empty_cuda(size, dt, dev, std::nullopt));
}
inline Tensor conform(const Tensor& t, at::ScalarType dt) {
  if (t.scalar_type() != dt) return t.to(dt).contiguous();
  return t.is_contiguous() ? t : t.contiguous();
}
inline Tensor f32c(const Tensor& t) { return t.defined() ? conform(t, at::kFloat) : t; }
inline const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline const float* fptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
inline float* fout(const Tensor& t) { return t.defined() ? static_cast<float*>(t.mutable_data_ptr()) : nullptr; }
inline void* current_stream(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

inline void check(int rc, const char* what) {
  if (rc == MLSTM_OK) return;
  std::string msg = std::string(what) + ": " + mlstm_b200_error_string(rc);
  if (rc == MLSTM_ERR_CUDA) TORCH_CHECK(false, msg, ": ", mlstm_b200_last_cuda_error());
  C10_THROW_ERROR(ValueError, msg);
}

inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }
inline Tensor bytes(size_t n, const at::Device& dev) { return empty({(int64_t)std::max<size_t>(n, 256)}, at::kByte, dev); }
// ---- Python arguments ------------------------------------------------------------------------------------
inline Tensor arg(PyObject* o, const char* name) {
  if (o == Py_None) return Tensor();
  if (!THPVariable_Check(o)) throw torch::TypeError(c10::str(name, " must be a tensor, got ", Py_TYPE(o)->tp_name));
  return THPVariable_Unpack(o);
}
inline Tensor need(PyObject* o, const char* name) {
  Tensor t = arg(o, name);
  if (!t.defined()) throw torch::TypeError(c10::str(name, " must be a tensor, got None"));
  return t;
}
inline at::ScalarType dtype_arg(PyObject* o) {
  if (!THPDtype_Check(o)) throw torch::TypeError(c10::str("expected a torch.dtype, got ", Py_TYPE(o)->tp_name));
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
inline PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
inline double double_arg(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}
inline long long_arg(PyObject* o) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}
inline bool bool_arg(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw python_error();
  return x != 0;
}
inline void nargs_are(Py_ssize_t have, Py_ssize_t want) {
  if (have != want) throw torch::TypeError(c10::str("expected ", want, " arguments, got ", have));
}

// host_layers.cpp: layer norm, short convolution, state space scan
extern PyMethodDef kLayerMethods[];

}  // namespace mlstm_host
