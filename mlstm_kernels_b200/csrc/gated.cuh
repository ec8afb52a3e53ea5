// The gates of the gated linear recurrence, shared by its forward, its backward and its step:
//
//   log a = log sigmoid(f), or rate sigmoid(f);   s = 1, 1 - a or sqrt(1 - a^2);   u = s sigmoid(i) x
//   h_t = a_t h_{t-1} + u_t;   y_t = h_t z_t sigmoid(z_t)
//
// 1 - a is computed by itself, with all of f32's digits but the last two, for the input's scale and the gradients, and a near one as
// 1 - (1 - a).  The state is multiplied by a as f32 has it, off by up to 2^-25, and joined runs by products of such factors, each off by as
// much: what a state forgets in a token is off by up to 2^-24 of the state, 2^-24 / (1 - a) of itself.  (A complement carried through
// the runs instead would leave the state's own rounding, 2^-24 of it in every join, and lose the digits of an a near zero.)
// All on pairs of values, for the packed instructions.
//
// Backward, with G_t = dL/dh_t (G_t = dy_t z_t sigmoid(z_t) + a_{t+1} G_{t+1}): everything that goes through a is
//
//   dL/d log a = G a w,   w = h_{t-1} - e,   e = 0, sigmoid(i) x, or a sigmoid(i) x / s     (s = 1, 1 - a, sqrt(1 - a^2))
//
// as a ds/da = -a or -a^2 / s; no quotient is left that a closed gate (1 - a = 0) would make 0 / 0.
#pragma once
#include "divide.cuh"
#include "gated_units.h"
#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

struct GatedDims {
  unsigned looks;       // how often a wait looks at memory, at most
  int S, D, nc;         // nc: kept states of a sequence
  int scale;
  int warps, nt, group, groups, units;   // (gated_units.h)
  Divide chains, blocks;
  long long xb, xt, fb, ft, ib, it, zb, zt, gb, gt;   // strides in elements (batch, token) of x, f, i, z, dy
  // scratch: null where a chain is one unit
  unsigned *ticket, *gave_up;
  uint2* state;
  uint4* agg;
};

template <typename T> struct GatedPtrs {
  const T *x, *f, *i, *z, *dy;
  const float *rate, *h0, *ckpt_in, *dh_last;
  T *y, *dx, *df, *di, *dz;
  float *h_last, *ckpt, *dh0, *rate_parts;
};

constexpr int GATED_PLAIN = 0, GATED_CONVEX = 1, GATED_VARIANCE = 2;

__device__ __forceinline__ float rsq(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint64_t dup2(float x) { return f2(x, x); }
__device__ __forceinline__ uint64_t minus2(uint64_t a, uint64_t b) { return fma2(b, dup2(-1.f), a); }   // a - b

template <typename T> __device__ __forceinline__ uint64_t logistic_pair2(uint64_t v) {
  float a, b;
  unf2(v, a, b);
  return logistic_pair<T>(a, b);
}

// s = sigmoid(v) and c = 1 - s of two values, both with all digits: whichever is above 1/2 is one minus the other
template <typename T> __device__ __forceinline__ void logistic_both(uint64_t v, uint64_t& s, uint64_t& c) {
  float v0, v1;
  unf2(v, v0, v1);
  const uint64_t e = exp_neg_pair<kFull<T>>(v0, v1), p = rcp_pair(add2(dup2(1.f), e)), q = mul2(e, p);
  // (where e is infinite, q is no number, and is not taken)
  float p0, p1, q0, q1, np0, np1, nq0, nq1;
  unf2(p, p0, p1);
  unf2(q, q0, q1);
  unf2(minus2(dup2(1.f), p), np0, np1);
  unf2(minus2(dup2(1.f), q), nq0, nq1);
  const bool up0 = v0 > 0.f, up1 = v1 > 0.f;
  s = f2(up0 ? nq0 : p0, up1 ? nq1 : p1);
  c = f2(up0 ? q0 : np0, up1 ? q1 : np1);
}

// The same where it is a gate: s by itself, c = e s, which keeps its digits wherever s is more than zero.  (Exponents end at 127, so
// that e stays a number; 1 / 2^127 is zero already, and what c is multiplied by then too.)
template <typename T> __device__ __forceinline__ void logistic_gate(uint64_t v, uint64_t& s, uint64_t& c) {
  float v0, v1;
  unf2(v, v0, v1);
  const uint64_t e = exp_neg_pair<kFull<T>>(max_nan(v0, -88.0296919f), max_nan(v1, -88.0296919f));
  s = rcp_pair(add2(dup2(1.f), e));
  c = mul2(e, s);
}

// of two values of f: a, 1 - a; and with a rate sigmoid(f) and 1 - sigmoid(f).
// FAR = false: the rate is known to be in (-1/2, 0], and no exponential is needed; BOTH = false: 1 - sigmoid(f) is not needed.
struct Decay { uint64_t a, rest, sf, cf; };
template <typename T, bool RATE, bool FAR = true, bool BOTH = true> __device__ __forceinline__ Decay decay_pair(uint64_t f, uint64_t rate) {
  Decay d;
  if constexpr (!RATE) {
    logistic_both<T>(f, d.sf, d.cf);
    d.a = d.sf;
    d.rest = d.cf;
    return d;
  }
  if constexpr (BOTH) logistic_gate<T>(f, d.sf, d.cf);
  else d.sf = logistic_pair2<T>(f);
  // l = log a = -rho.  Where rho is below 1/2: 1 - e^l = rho p(l), p the polynomial through the values of (e^l - 1) / l at the
  // Chebyshev points of [-1/2, 0], off by 2^-29, in f32 2^-24; else 1 - a has lost one digit at most.
  const uint64_t l = mul2(rate, d.sf), rho = mul2(l, dup2(-1.f));
  uint64_t p = fma2(dup2(1.1234042e-3f), l, dup2(8.1896136e-3f));
  p = fma2(p, l, dup2(4.1630073e-2f));
  p = fma2(p, l, dup2(1.6666242e-1f));
  p = fma2(p, l, dup2(4.9999982e-1f));
  p = fma2(p, l, dup2(1.f));
  const uint64_t small = mul2(p, rho), large = fma2(p, l, dup2(1.f));
  if constexpr (!FAR) {
    d.rest = small;
    d.a = large;
    return d;
  }
  float r0, r1, s0, s1, l0, l1, e0, e1;
  unf2(rho, r0, r1);
  unf2(small, s0, s1);
  unf2(large, l0, l1);
  unf2(exp_neg_pair<kFull<T>>(r0, r1), e0, e1);
  const bool n0 = __float_as_uint(r0) < 0x3f000000u, n1 = __float_as_uint(r1) < 0x3f000000u;   // (0 <= rho < 1/2)
  d.rest = f2(n0 ? s0 : 1.f - e0, n1 ? s1 : 1.f - e1);
  d.a = f2(n0 ? l0 : e0, n1 ? l1 : e1);
  return d;
}

// 1 / sqrt(1 - a^2), finite where a = 1 (what it is multiplied by is zero then)
__device__ __forceinline__ uint64_t inv_scale_pair(uint64_t rest2) {
  float q0, q1;
  unf2(add2(rest2, dup2(1.17549435e-38f)), q0, q1);
  return f2(rsq(q0), rsq(q1));
}
__device__ __forceinline__ uint64_t rest2_pair(uint64_t a, uint64_t rest) { return fma2(rest, a, rest); }   // 1 - a^2

// What is there, known when a kernel is called
struct GatedAny {
  bool rate_, i_, z_;
  int scale_;
  __device__ bool rate() const { return rate_; }
  __device__ int scale() const { return scale_; }
  __device__ bool i() const { return i_; }
  __device__ bool z() const { return z_; }
};

// ---- runs of tokens ---------------------------------------------------------------------------------
struct Run { uint64_t A, H; };   // of two channels
__device__ __forceinline__ Run no_tokens() { return Run{dup2(1.f), 0}; }
__device__ __forceinline__ Run then(Run first, Run second) { return Run{mul2(second.A, first.A), fma2(second.A, first.H, second.H)}; }
__device__ __forceinline__ uint64_t through(Run r, uint64_t h) { return fma2(r.A, h, r.H); }

// FAR: the rate may be outside (-1/2, 0]
template <typename T, bool FAR, bool BOTH, class M> __device__ __forceinline__ Decay gated_decay(const M& m, uint64_t f, uint64_t rate) {
  if (m.rate()) return decay_pair<T, true, FAR, BOTH>(f, rate);
  return decay_pair<T, false>(f, rate);
}
__device__ __forceinline__ bool far_rate(uint64_t rate) {
  float r0, r1;
  unf2(rate, r0, r1);
  return !(r0 > -0.5f && r0 <= 0.f && r1 > -0.5f && r1 <= 0.f);
}

// ---- one token of a pair of channels ------------------------------------------------------------------
// Forward: its factor, and what it adds
template <typename T, bool FAR, class M> __device__ __forceinline__ Run gated_token(const M& m, uint64_t f, uint64_t x, uint64_t i, uint64_t rate) {
  const Decay d = gated_decay<T, FAR, false>(m, f, rate);
  uint64_t u = x;
  if (m.i()) u = mul2(u, logistic_pair2<T>(i));
  if (m.scale() == GATED_CONVEX) u = mul2(u, d.rest);
  if (m.scale() == GATED_VARIANCE) {
    const uint64_t q2 = rest2_pair(d.a, d.rest);
    u = mul2(mul2(u, q2), inv_scale_pair(q2));
  }
  return Run{d.a, u};
}

}  // namespace mlstm
