// Gated linear recurrence (formulas: gated.cuh): forward, backward, and the step for one token.
// One thread to a channel of a sequence, token after token; the backward takes GATED_CK tokens at a time, last ones first, and
// recomputes their states from the one before them, which the forward has kept.
#include "gated.cuh"

namespace mlstm {

constexpr int GATED_CK = 8;

struct GatedDims {
  int B, S, D, nc;   // nc: kept states
  int scale;
  long long xb, xt, fb, ft, ib, it, zb, zt, gb, gt;   // strides in elements (batch, token) of x, f, i, z, dy
};

// one token of one channel
template <typename T, bool RATE> struct GatedToken {
  float a, rest, sf, cf, g, cg, x, s, rs;   // sigmoid(i) and one minus it; the input's scale and 1 / sqrt(1 - a^2)
  __device__ GatedToken(const T* x_, const T* f_, const T* i_, float rate, int scale) {
    x = to_f32(*x_);
    const float f = to_f32(*f_);
    const Decay d = decay_pair<T, RATE>(f2(f, f), f2(rate, rate));
    float o;
    unf2(d.a, a, o);
    unf2(d.rest, rest, o);
    unf2(d.sf, sf, o);
    unf2(d.cf, cf, o);
    g = 1.f, cg = 0.f;
    if (i_ != nullptr) {
      const float i = to_f32(*i_);
      uint64_t gp, cp;
      logistic_both<T>(f2(i, i), gp, cp);
      unf2(gp, g, o);
      unf2(cp, cg, o);
    }
    const uint64_t q = rest2_pair(d.a, d.rest), r = inv_scale_pair(q);
    float qq;
    unf2(q, qq, o);
    unf2(r, rs, o);
    s = scale == GATED_PLAIN ? 1.f : scale == GATED_CONVEX ? rest : qq * rs;
  }
};

template <typename T, bool RATE>
__global__ void gated_fw(const T* x, const T* f, const T* i, const T* z, const float* rate, const float* h0, T* y, float* h_last, float* ckpt, GatedDims q) {
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= (long long)q.B * q.D) return;
  const int b = (int)(n / q.D), d = (int)(n % q.D);
  const float r = RATE ? rate[d] : 0.f;
  float h = h0 != nullptr ? h0[n] : 0.f;
  for (int t = 0; t < q.S; ++t) {
    if (ckpt != nullptr && t % GATED_CK == 0) ckpt[((long long)b * q.nc + t / GATED_CK) * q.D + d] = h;
    const GatedToken<T, RATE> k(x + b * q.xb + t * q.xt + d, f + b * q.fb + t * q.ft + d, i != nullptr ? i + b * q.ib + t * q.it + d : nullptr, r, q.scale);
    h = k.a * h + k.s * k.g * k.x;
    float out = h;
    if (z != nullptr) {
      const float zz = to_f32(z[b * q.zb + t * q.zt + d]);
      out *= zz * logistic_f<T>(zz);
    }
    y[((long long)b * q.S + t) * q.D + d] = from_f32<T>(out);
  }
  if (h_last != nullptr) h_last[n] = h;
}

template <typename T, bool RATE>
__global__ void gated_bw(const T* x, const T* f, const T* i, const T* z, const float* rate, const float* ckpt, const T* dy, const float* dh_last, T* dx,
                         T* df, T* di, T* dz, float* drate, float* dh0, GatedDims q) {
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= (long long)q.B * q.D) return;
  const int b = (int)(n / q.D), d = (int)(n % q.D);
  const float r = RATE ? rate[d] : 0.f;
  float c = dh_last != nullptr ? dh_last[n] : 0.f, dr = 0.f;   // c: a_{t+1} G_{t+1}
  auto token = [&](int t) {
    return GatedToken<T, RATE>(x + b * q.xb + t * q.xt + d, f + b * q.fb + t * q.ft + d, i != nullptr ? i + b * q.ib + t * q.it + d : nullptr, r, q.scale);
  };
  for (int k0 = q.nc - 1; k0 >= 0; --k0) {
    float before[GATED_CK + 1];
    before[0] = ckpt[((long long)b * q.nc + k0) * q.D + d];
#pragma unroll
    for (int j = 0; j < GATED_CK; ++j) {
      const int t = k0 * GATED_CK + j;
      if (t < q.S) {
        const GatedToken<T, RATE> k = token(t);
        before[j + 1] = k.a * before[j] + k.s * k.g * k.x;
      }
    }
#pragma unroll
    for (int j = GATED_CK - 1; j >= 0; --j) {
      const int t = k0 * GATED_CK + j;
      if (t >= q.S) continue;
      const long long at = ((long long)b * q.S + t) * q.D + d;
      const GatedToken<T, RATE> k = token(t);
      float up = to_f32(dy[b * q.gb + t * q.gt + d]);
      if (z != nullptr) {
        const float zz = to_f32(z[b * q.zb + t * q.zt + d]);
        uint64_t sp, cp;
        logistic_both<T>(f2(zz, zz), sp, cp);
        float s, cs, o;
        unf2(sp, s, o);
        unf2(cp, cs, o);
        dz[at] = from_f32<T>(up * before[j + 1] * (s * (1.f + zz * cs)));
        up *= zz * s;
      }
      const float G = up + c, gx = k.g * k.x;
      const float w = before[j] - (q.scale == GATED_PLAIN ? 0.f : q.scale == GATED_CONVEX ? gx : k.a * gx * k.rs);
      c = k.a * G;
      dx[at] = from_f32<T>(G * k.s * k.g);
      if (di != nullptr) di[at] = from_f32<T>(G * k.s * gx * k.cg);
      if constexpr (RATE) {
        const float base = c * w * k.sf;   // of the rate
        df[at] = from_f32<T>(base * r * k.cf);
        dr += base;
      } else {
        df[at] = from_f32<T>(c * w * k.rest);
      }
    }
  }
  if (dh0 != nullptr) dh0[n] = c;
  if (RATE && drate != nullptr) drate[n] = dr;
}

__global__ void gated_rate_sum(const float* parts, float* drate, int n, int D) {
  const int d = blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= D) return;
  float s = 0.f;
  for (int k = 0; k < n; ++k) s += parts[(long long)k * D + d];
  drate[d] = s;
}

template <typename T, bool RATE>
__global__ void gated_one(const T* x, const T* f, const T* i, const T* z, const float* rate, const float* h, T* y, float* h_new, long long n, int D, int scale) {
  const long long k = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (k >= n) return;
  const GatedToken<T, RATE> t(x + k, f + k, i != nullptr ? i + k : nullptr, RATE ? rate[k % D] : 0.f, scale);
  const float v = t.a * h[k] + t.s * t.g * t.x;
  h_new[k] = v;
  float out = v;
  if (z != nullptr) {
    const float zz = to_f32(z[k]);
    out *= zz * logistic_f<T>(zz);
  }
  y[k] = from_f32<T>(out);
}

bool gated_sizes_ok(int B, int S, int D) { return B > 0 && S > 0 && D > 0 && (long long)B * D <= (1ll << 40); }
size_t gated_ckpt_bytes(int B, int S, int D) { return (size_t)B * ceil_div(S, GATED_CK) * D * sizeof(float); }
size_t gated_bw_bytes(int B, int S, int D) { return (size_t)B * D * sizeof(float); }

static GatedDims gated_dims(const long long* st, int B, int S, int D, int scale) {
  return GatedDims{B, S, D, ceil_div(S, GATED_CK), scale, st[0], st[1], st[2], st[3], st[4], st[5], st[6], st[7], 0, 0};
}

int launch_gated_fw(const GatedIn& in, const long long* strides, void* y, float* h_last, float* ckpt, int B, int S, int D, int scale, int dtype,
                    cudaStream_t st) {
  PhaseScope ps(PH_GATED, st);
  const GatedDims q = gated_dims(strides, B, S, D, scale);
  const unsigned grid = (unsigned)(((long long)B * D + 127) / 128);
  auto go = [&](auto* t, auto rate) {
    using T = std::remove_pointer_t<decltype(t)>;
    gated_fw<T, decltype(rate)::value><<<grid, 128, 0, st>>>((const T*)in.x, (const T*)in.f, (const T*)in.i, (const T*)in.z, in.rate, in.h0, (T*)y, h_last,
                                                               ckpt, q);
  };
  MLSTM_DTYPE_SWITCH(dtype, T, if (in.rate != nullptr) go((T*)nullptr, std::true_type{}); else go((T*)nullptr, std::false_type{});)
  MLSTM_LAUNCH_CHECK();
  return MLSTM_OK;
}

int launch_gated_bw(const GatedIn& in, const long long* strides, const float* ckpt, const void* dy, const long long* gs, const float* dh_last, void* dx,
                    void* df, void* di, void* dz, float* drate, float* dh0, float* parts, int B, int S, int D, int scale, int dtype, cudaStream_t st) {
  PhaseScope ps(PH_GATED, st);
  GatedDims q = gated_dims(strides, B, S, D, scale);
  q.gb = gs[0], q.gt = gs[1];
  const unsigned grid = (unsigned)(((long long)B * D + 127) / 128);
  auto go = [&](auto* t, auto rate) {
    using T = std::remove_pointer_t<decltype(t)>;
    gated_bw<T, decltype(rate)::value><<<grid, 128, 0, st>>>((const T*)in.x, (const T*)in.f, (const T*)in.i, (const T*)in.z, in.rate, ckpt, (const T*)dy,
                                                               dh_last, (T*)dx, (T*)df, (T*)di, (T*)dz, drate != nullptr ? parts : nullptr, dh0, q);
  };
  MLSTM_DTYPE_SWITCH(dtype, T, if (in.rate != nullptr) go((T*)nullptr, std::true_type{}); else go((T*)nullptr, std::false_type{});)
  MLSTM_LAUNCH_CHECK();
  if (drate != nullptr) {
    gated_rate_sum<<<ceil_div(D, 128), 128, 0, st>>>(parts, drate, B, D);
    MLSTM_LAUNCH_CHECK();
  }
  return MLSTM_OK;
}

int launch_gated_step(const GatedIn& in, const float* h, void* y, float* h_new, int B, int D, int scale, int dtype, cudaStream_t st) {
  PhaseScope ps(PH_GATED, st);
  const long long n = (long long)B * D;
  const unsigned grid = (unsigned)((n + 127) / 128);
  auto go = [&](auto* t, auto rate) {
    using T = std::remove_pointer_t<decltype(t)>;
    gated_one<T, decltype(rate)::value><<<grid, 128, 0, st>>>((const T*)in.x, (const T*)in.f, (const T*)in.i, (const T*)in.z, in.rate, h, (T*)y, h_new, n,
                                                                D, scale);
  };
  MLSTM_DTYPE_SWITCH(dtype, T, if (in.rate != nullptr) go((T*)nullptr, std::true_type{}); else go((T*)nullptr, std::false_type{});)
  MLSTM_LAUNCH_CHECK();
  return MLSTM_OK;
}

}  // namespace mlstm
