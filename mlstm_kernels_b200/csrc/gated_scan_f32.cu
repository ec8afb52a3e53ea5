// The gated linear recurrence of f32 tensors.
#include "gated_tiles.cuh"

namespace mlstm {
int gated_run_f32(bool back, bool rows, const void* ptrs, const GatedDims& q, cudaStream_t st) {
  return gated_run<float>(back, rows, *static_cast<const GatedPtrs<float>*>(ptrs), q, st);
}
int gated_status_f32(int reset, int* status) { return gated_status_of(reset, status); }
}  // namespace mlstm
