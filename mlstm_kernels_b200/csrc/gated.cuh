// The gates of the gated linear recurrence, shared by its forward, its backward and its step:
//
//   log a = log sigmoid(f), or rate sigmoid(f);   s = 1, 1 - a or sqrt(1 - a^2);   u = s sigmoid(i) x
//   h_t = a_t h_{t-1} + u_t;   y_t = h_t z_t sigmoid(z_t)
//
// What a long recurrence remembers hangs on 1 - a: it is computed by itself, with all of f32's digits but the last two, and a near
// one as 1 - (1 - a).  All on pairs of values, for the packed instructions.
//
// Backward, with G_t = dL/dh_t (G_t = dy_t z_t sigmoid(z_t) + a_{t+1} G_{t+1}): everything that goes through a is
//
//   dL/d log a = G a w,   w = h_{t-1} - e,   e = 0, sigmoid(i) x, or a sigmoid(i) x / s     (s = 1, 1 - a, sqrt(1 - a^2))
//
// as a ds/da = -a or -a^2 / s; no quotient is left that a closed gate (1 - a = 0) would make 0 / 0.
#pragma once
#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

constexpr int GATED_CK = 8;   // tokens to a thread, and to a state that the forward keeps for the backward
struct GatedDims {
  int B, S, D, nc;      // nc: kept states of a sequence
  int scale;
  int blocks;           // CTAs next to each other that take the channels
  int K, warps;         // CTAs to a cluster, warps to a CTA
  long long xb, xt, fb, ft, ib, it, zb, zt, gb, gt;   // strides in elements (batch, token) of x, f, i, z, dy
};

constexpr int GATED_PLAIN = 0, GATED_CONVEX = 1, GATED_VARIANCE = 2;

__device__ __forceinline__ float rsq(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint64_t dup2(float x) { return f2(x, x); }
__device__ __forceinline__ uint64_t neg2(uint64_t v) { return v ^ 0x8000000080000000ull; }

// s = sigmoid(v) and c = 1 - s of two values, both with all digits: whichever is above 1/2 is one minus the other
template <typename T> __device__ __forceinline__ void logistic_both(uint64_t v, uint64_t& s, uint64_t& c) {
  float v0, v1;
  unf2(v, v0, v1);
  const uint64_t e = exp_neg_pair<kFull<T>>(v0, v1), p = rcp_pair(add2(dup2(1.f), e)), q = mul2(e, p);
  // (where e is infinite, q is no number, and is not taken)
  float p0, p1, q0, q1;
  unf2(p, p0, p1);
  unf2(q, q0, q1);
  const float less0 = v0 > 0.f ? q0 : p0, less1 = v1 > 0.f ? q1 : p1, more0 = 1.f - less0, more1 = 1.f - less1;
  s = f2(v0 > 0.f ? more0 : less0, v1 > 0.f ? more1 : less1);
  c = f2(v0 > 0.f ? less0 : more0, v1 > 0.f ? less1 : more1);
}

// of two values of f: a, 1 - a; and with a rate sigmoid(f) and 1 - sigmoid(f)
struct Decay { uint64_t a, rest, sf, cf; };
// (FAR = false: the rate is known to be in (-1/2, 0], and no exponential is needed)
template <typename T, bool RATE, bool FAR = true> __device__ __forceinline__ Decay decay_pair(uint64_t f, uint64_t rate) {
  Decay d;
  logistic_both<T>(f, d.sf, d.cf);
  if constexpr (!RATE) {
    d.a = d.sf;
    d.rest = d.cf;
  } else {
    // rho = -log a.  Below 1/2: 1 - e^-rho = rho p(rho), p the polynomial through its values at the Chebyshev points of [0, 1/2],
    // off by 2^-29, in f32 2^-24; else 1 - a has lost one digit at most.
    const uint64_t rho = neg2(mul2(rate, d.sf));
    uint64_t p = fma2(dup2(-1.1234042e-3f), rho, dup2(8.1896136e-3f));
    p = fma2(p, rho, dup2(-4.1630073e-2f));
    p = fma2(p, rho, dup2(1.6666242e-1f));
    p = fma2(p, rho, dup2(-4.9999982e-1f));
    p = fma2(p, rho, dup2(1.f));
    const uint64_t small = mul2(p, rho);
    if constexpr (!FAR) {
      d.rest = small;
      d.a = fma2(p, neg2(rho), dup2(1.f));
      return d;
    }
    float r0, r1, s0, s1, e0, e1;
    unf2(rho, r0, r1);
    unf2(small, s0, s1);
    unf2(exp_neg_pair<kFull<T>>(r0, r1), e0, e1);
    const bool n0 = __float_as_uint(r0) < 0x3f000000u, n1 = __float_as_uint(r1) < 0x3f000000u;   // (0 <= rho < 1/2)
    const float rest0 = n0 ? s0 : 1.f - e0, rest1 = n1 ? s1 : 1.f - e1;
    d.rest = f2(rest0, rest1);
    d.a = f2(n0 ? 1.f - s0 : e0, n1 ? 1.f - s1 : e1);
  }
  return d;
}

// 1 / sqrt(1 - a^2), finite where a = 1 (what it is multiplied by is zero then)
__device__ __forceinline__ uint64_t inv_scale_pair(uint64_t rest2) {
  float q0, q1;
  unf2(add2(rest2, dup2(1.17549435e-38f)), q0, q1);
  return f2(rsq(q0), rsq(q1));
}
__device__ __forceinline__ uint64_t rest2_pair(uint64_t a, uint64_t rest) { return fma2(rest, a, rest); }   // 1 - a^2

template <typename T> __device__ __forceinline__ uint64_t logistic_pair2(uint64_t v) {
  float a, b;
  unf2(v, a, b);
  return logistic_pair<T>(a, b);
}

}  // namespace mlstm
