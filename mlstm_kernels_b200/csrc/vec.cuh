// Several neighbouring elements in one access, and parameters whose element type is known at run time only.
#pragma once
#include "common.cuh"

namespace mlstm {

// V elements of T as they lie in memory; V * sizeof(T) <= 16 is one access, more is several of 16 bytes.
template <typename T, int V> struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack { T e[V]; };

template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) { *reinterpret_cast<Pack<T, V>*>(p) = v; }
template <typename T, int V> __device__ __forceinline__ Pack<T, V> zero_pack() {
  Pack<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.e[i] = from_f32<T>(0.f);
  return v;
}

__device__ __forceinline__ float load_any(const void* p, size_t idx, int dtype) {
  if (dtype == MLSTM_F32) return static_cast<const float*>(p)[idx];
  if (dtype == MLSTM_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[idx]);
  return to_f32(static_cast<const __half*>(p)[idx]);
}
__device__ __forceinline__ void store_any(void* p, size_t idx, float x, int dtype) {
  if (dtype == MLSTM_F32) static_cast<float*>(p)[idx] = x;
  else if (dtype == MLSTM_BF16) static_cast<__nv_bfloat16*>(p)[idx] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[idx] = __float2half_rn(x);
}
// V of them that follow one another from an index that is a multiple of V, at a base aligned to 16 bytes
template <int V> __device__ __forceinline__ void load_any(const void* p, size_t idx, int dtype, float (&o)[V]) {
  if (V > 1 && dtype == MLSTM_F32) {
    const Pack<float, V> v = load_pack<float, V>(static_cast<const float*>(p) + idx);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = v.e[i];
  } else if (V > 1 && dtype == MLSTM_BF16) {
    const Pack<__nv_bfloat16, V> v = load_pack<__nv_bfloat16, V>(static_cast<const __nv_bfloat16*>(p) + idx);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f32(v.e[i]);
  } else if (V > 1) {
    const Pack<__half, V> v = load_pack<__half, V>(static_cast<const __half*>(p) + idx);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f32(v.e[i]);
  } else {
    o[0] = load_any(p, idx, dtype);
  }
}

// Host: may rows at these offsets (in elements) from p be accessed `bytes` at a time?
inline bool fits_access(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool stride_fits(long long elements, size_t element_size, size_t bytes) { return (elements * (long long)element_size) % (long long)bytes == 0; }

#define MLSTM_DTYPE_SWITCH(code, T, ...)                                            \
  switch (code) {                                                                   \
    case MLSTM_F32: { using T = float; __VA_ARGS__ } break;                         \
    case MLSTM_BF16: { using T = __nv_bfloat16; __VA_ARGS__ } break;                \
    case MLSTM_F16: { using T = __half; __VA_ARGS__ } break;                        \
  }

}  // namespace mlstm
