// The gated linear recurrence of f16 tensors.
#include "gated_tiles.cuh"

namespace mlstm {
int gated_run_f16(bool back, bool rows, const void* ptrs, const GatedDims& q, cudaStream_t st) {
  return gated_run<__half>(back, rows, *static_cast<const GatedPtrs<__half>*>(ptrs), q, st);
}
int gated_status_f16(int reset, int* status) { return gated_status_of(reset, status); }
}  // namespace mlstm
