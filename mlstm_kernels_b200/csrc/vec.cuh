// Several neighbouring elements in one access, and parameters whose element type is known at run time only.
#pragma once
#include "common.cuh"
#include "f32x2.cuh"

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

// ---- asynchronous copies ------------------------------------------------------------------------------
// V elements to shared memory: they arrive by a later cp_wait(), zeros where `ok` is false (the address must exist even so).
// Accesses below four bytes, which cannot be asynchronous, are made at once.
template <typename T, int V> __device__ __forceinline__ void copy_async(T* dst, const T* src, bool ok) {
  constexpr int BYTES = sizeof(T) * V;
  if constexpr (BYTES >= 4) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(BYTES), "r"(ok ? BYTES : 0) : "memory");
  } else {
    store_pack<T, V>(dst, ok ? load_pack<T, V>(src) : zero_pack<T, V>());
  }
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- exponentials for element-wise work ----------------------------------------------------------------
// The hardware's 2^x and 1 / x, off by 2^-22 and 2^-23 of the result (results below 2^-126 are zero), instead of expf and a
// division, which take thirty instructions.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = (float)(1.4426950408889634 - (double)kLog2e), kLn2 = 0.6931471805599453f;
__device__ __forceinline__ uint64_t ex2_pair(uint64_t v) {
  float a, b;
  unf2(v, a, b);
  return f2(ex2(a), ex2(b));
}
__device__ __forceinline__ uint64_t rcp_pair(uint64_t v) {
  float a, b;
  unf2(v, a, b);
  return f2(rcp(a), rcp(b));
}
// e^-x of two values.  FULL: what the rounding of x log2(e) dropped, r, is put back, 2^(n + r) = 2^n (1 + r ln 2): all of f32's digits
// but the last two.  Without, the result is off by 1.5 |x| 2^-24 of itself (x = 60: 5e-6): for results that are rounded to 16 bits
// next, and for steps, where a dt in 16 bits is off by 2^-12 |x| and more to begin with (put back there too, a training step of the
// scan of 4 x 2048 x 2048 x 16 in bf16 takes 748 us instead of 736).
template <bool FULL> __device__ __forceinline__ uint64_t exp_neg_pair(float x0, float x1) {
  if constexpr (!FULL) return ex2_pair(mul2(f2(x0, x1), f2(-kLog2e, -kLog2e)));
  // (beyond +-1e4 as there: zero and infinity; r must stay a number)
  const uint64_t x = f2(min_nan(max_nan(x0, -1e4f), 1e4f), min_nan(max_nan(x1, -1e4f), 1e4f)), n = mul2(x, f2(-kLog2e, -kLog2e));
  const uint64_t r = fma2(x, f2(-kLog2eRest, -kLog2eRest), fma2(x, f2(-kLog2e, -kLog2e), mul2(x, f2(kLog2e, kLog2e))));
  return mul2(ex2_pair(n), fma2(r, f2(kLn2, kLn2), f2(1.f, 1.f)));
}
// Element types of inputs and results that keep f32's digits
template <typename T> constexpr bool kFull = sizeof(T) == 4;
template <typename T> __device__ __forceinline__ uint64_t logistic_pair(float x0, float x1) {
  return rcp_pair(add2(f2(1.f, 1.f), exp_neg_pair<kFull<T>>(x0, x1)));
}
template <typename T> __device__ __forceinline__ float logistic_f(float x) {
  if constexpr (!kFull<T>) return rcp(1.f + ex2(-kLog2e * x));
  float a, b;
  unf2(logistic_pair<T>(x, x), a, b);
  return a;
}
// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x|; log(1 + e) = 2 artanh(s), s = e / (2 + e) <= 1/3, which keeps all digits of a
// small e.  artanh(s) / s as a polynomial in s^2, through its values at the Chebyshev points of [0, 1/9]: off by 2^-26.
template <typename T> __device__ __forceinline__ uint64_t softplus_pair(float x0, float x1) {
  const uint64_t e = exp_neg_pair<kFull<T>>(fabsf(x0), fabsf(x1));
  const uint64_t s = mul2(e, rcp_pair(add2(e, f2(2.f, 2.f)))), q = mul2(s, s);
  uint64_t p = fma2(f2(0.14078890f, 0.14078890f), q, f2(0.13982579f, 0.13982579f));
  p = fma2(p, q, f2(0.20012298f, 0.20012298f));
  p = fma2(p, q, f2(0.33333161f, 0.33333161f));
  p = fma2(p, q, f2(1.f, 1.f));
  return fma2(add2(s, s), p, f2(max_nan(x0, 0.f), max_nan(x1, 0.f)));
}
template <typename T, int V> __device__ __forceinline__ void logistic_v(const float (&x)[V], float (&o)[V]) {
  if constexpr (V == 1) {
    o[0] = logistic_f<T>(x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) unf2(logistic_pair<T>(x[i], x[i + 1]), o[i], o[i + 1]);
  }
}
template <typename T, int V> __device__ __forceinline__ void softplus_v(const float (&x)[V], float (&o)[V]) {
  if constexpr (V == 1) {
    float other;
    unf2(softplus_pair<T>(x[0], x[0]), o[0], other);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) unf2(softplus_pair<T>(x[i], x[i + 1]), o[i], o[i + 1]);
  }
}
template <typename T, int V> __device__ __forceinline__ void unpack(const Pack<T, V>& p, float (&o)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = to_f32(p.e[i]);
}
// (two 16-bit elements to a conversion)
__device__ __forceinline__ void from_f32x2(float a, float b, float* o) { o[0] = a; o[1] = b; }
__device__ __forceinline__ void from_f32x2(float a, float b, __nv_bfloat16* o) { *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ void from_f32x2(float a, float b, __half* o) { *reinterpret_cast<__half2*>(o) = __floats2half2_rn(a, b); }
template <typename T, int V> __device__ __forceinline__ Pack<T, V> pack(const float (&o)[V]) {
  Pack<T, V> p;
  if constexpr (V == 1) {
    p.e[0] = from_f32<T>(o[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) from_f32x2(o[i], o[i + 1], p.e + i);
  }
  return p;
}

#define MLSTM_DTYPE_SWITCH(code, T, ...)                                            \
  switch (code) {                                                                   \
    case MLSTM_F32: { using T = float; __VA_ARGS__ } break;                         \
    case MLSTM_BF16: { using T = __nv_bfloat16; __VA_ARGS__ } break;                \
    case MLSTM_F16: { using T = __half; __VA_ARGS__ } break;                        \
  }

}  // namespace mlstm
