// What the host sides of the operators around a recurrence share: checks of their arguments, and tensors as their kernels read them.
#pragma once
#include "host.h"

namespace mlstm_host {

using OptT = std::optional<Tensor>;
inline OptT given(const Tensor& t) { return t.defined() ? OptT(t) : std::nullopt; }
inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// All on the device of the first; no forward-mode tangents, which would be dropped without a word.
inline void check_tensors(const char* op, std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), kNeedsCuda);
    if (t->device() != first.device()) C10_THROW_ERROR(ValueError, c10::str(op, ": tensors on different devices (", first.device(), " and ", t->device(), ")"));
    if (t->layout() != at::kStrided) C10_THROW_ERROR(ValueError, c10::str(op, ": tensors must be dense"));
    if (t->_fw_grad(0).defined()) C10_THROW_ERROR(NotImplementedError, c10::str("mlstm_kernels_b200 has no forward-mode derivative of ", op));
  }
}
inline void check_kernel_dtype(const Tensor& t) {
  if (t.defined() && dtype_code(t.scalar_type()) < 0) C10_THROW_ERROR(ValueError, c10::str("Unsupported kernel dtype ", t.dtype(), "."));
}
[[noreturn]] inline void bad_shape(const char* op, const char* name, const Tensor& t, const char* want) {
  C10_THROW_ERROR(ValueError, c10::str(op, ": ", name, " of shape ", t.sizes(), " must be ", want));
}
inline void check_int_sizes(const char* op, const Tensor& t) {   // the kernels count single axes in 32 bits
  for (const int64_t n : t.sizes())
    if (n > (1ll << 30)) C10_THROW_ERROR(ValueError, c10::str(op, ": an axis of more than 2^30 elements"));
}
inline void no_second_derivative(const char* op) {
  if (at::GradMode::is_enabled()) C10_THROW_ERROR(NotImplementedError, c10::str("mlstm_kernels_b200 has no second derivative of ", op));
}
// A buffer that a step writes (contiguous, as are those that it reads): it may be the state that it replaces, and lies apart from
// everything else.  Autograd is told of the write, so that a graph that kept the old contents does not take the new ones for them.
inline void check_written(const char* op, const char* name, const Tensor& out, const Tensor& state, std::initializer_list<const Tensor*> ins) {
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.const_data_ptr());
  auto meets = [&](const Tensor& t) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    return p < o + out.nbytes() && o < p + t.nbytes();
  };
  bool apart = state.const_data_ptr() == out.const_data_ptr() || !meets(state);
  for (const Tensor* t : ins) apart = apart && !(t->defined() && meets(*t));
  if (!apart) C10_THROW_ERROR(ValueError, c10::str(op, ": ", name, " overlaps a tensor that the step reads (only the whole old state may be replaced in place)"));
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}
// What a backward operator is given beside the forward's inputs
inline void check_size(const char* op, const char* name, const Tensor& t, at::IntArrayRef size) {
  if (t.defined() && t.sizes() != size) C10_THROW_ERROR(ValueError, c10::str(op, ": ", name, " of shape ", t.sizes(), " must be of shape ", size));
}
// as a kernel reads it: the last axis contiguous
inline Tensor last_dense(const Tensor& t) { return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
inline Tensor zeros(at::IntArrayRef size, at::ScalarType dt, const at::Device& dev) { return empty(size, dt, dev).zero_(); }
inline Tensor to_dtype(const Tensor& t, at::ScalarType dt) { return !t.defined() || t.scalar_type() == dt ? t : t.to(dt); }

// the stride of the token axis; of a single token any number will do
inline long long token_stride(const Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }
inline Tensor tokens_near(const Tensor& t) {   // the scan takes token strides below 2^29
  const Tensor d = last_dense(t);
  return !d.defined() || token_stride(d) < (1ll << 29) ? d : d.clone(at::MemoryFormat::Contiguous);
}

}  // namespace mlstm_host
