// The gated linear recurrence of bf16 tensors.
#include "gated_tiles.cuh"

namespace mlstm {
int gated_run_bf16(bool back, bool rows, const void* ptrs, const GatedDims& q, cudaStream_t st) {
  return gated_run<__nv_bfloat16>(back, rows, *static_cast<const GatedPtrs<__nv_bfloat16>*>(ptrs), q, st);
}
int gated_status_bf16(int reset, int* status) { return gated_status_of(reset, status); }
}  // namespace mlstm
