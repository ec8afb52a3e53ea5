// Selective state space scan, forward, and its step for one token.
//
//   step_t = softplus(dt_t + dt_bias) (or dt_t + dt_bias);   h_t[n] = exp(step_t a[n]) h_{t-1}[n] + step_t x_t b_t[n]
//   y_t = (sum_n c_t[n] h_t[n] + skip x_t) z_t sigmoid(z_t)          for every channel of its own, n = 0 ... N - 1
//
// Bound by the special function units: N exponentials a token and channel (16 a clock and SM) against 8 bytes of operands.  The
// states stay in f32 registers; a tile's steps and step * x are computed once, by all threads, and reach the recurrence through
// shared memory, and the sums over the states leave the same way.  Few sequences of few channels are cut into segments: each
// segment's end state from an empty start first (with the sum of its steps, whose exponential is its decay), then all segments at
// once, each folding what the ones before it left; twice the exponentials, on as many more SMs.
#include "ssm.cuh"

namespace mlstm {

struct SsmFw {
  SsmIn in;
  void* y;
  float* h_last;       // (B, D, N) or null
  float* ckpt;         // (B, nt, D, NP): the state before every tile, or null
  float* loc_h;        // (B, nseg, D, NP) end states of the segments, from an empty start
  float* loc_sum;      // (B, nseg, D) sums of their steps
};

// The state before segment p.seg
template <int LN, int V>
__device__ __forceinline__ void ssm_enter(const SsmFw& k, const SsmDims& s, const SsmPlace<LN, V>& p, const float (&a2)[4], float (&h)[4]) {
  constexpr int NP = 4 * LN;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = k.in.h0 != nullptr && p.on && 4 * p.sub + i < s.N ? k.in.h0[((size_t)p.b * s.D + p.d) * s.N + 4 * p.sub + i] : 0.f;
  if (!p.on) return;
  for (int j = 0; j < p.seg; ++j) {
    const size_t at = ((size_t)p.b * s.nseg + j) * s.D + p.d;
    const float sum = k.loc_sum[at];
    const Pack<float, 4> l = load_pack<float, 4>(k.loc_h + at * NP + 4 * p.sub);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = fmaf(ex2(sum * a2[i]), h[i], l.e[i]);
  }
}

// LOCAL: only a segment's own end state and sum of steps
template <typename T, int LN, int V, bool LOCAL>
__global__ void __launch_bounds__(SSM_THREADS, 3)
ssm_fw_kernel(SsmFw k, SsmDims s) {
  using P = SsmPlace<LN, V>;
  constexpr int CH = P::CH, NP = P::NP, TB = LN < 8 ? LN : 8;
  __shared__ float2 s_d[SSM_TT * CH];                          // (step, step x)
  __shared__ __align__(16) float s_b[SSM_TT * NP];
  __shared__ __align__(16) float s_c[LOCAL ? 4 : SSM_TT * NP];
  __shared__ __align__(16) float s_y[LOCAL ? 4 : SSM_TT * P::YS];
  pdl_launch_dependents();
  pdl_wait();
  const P p(s);
  float a2[4], h[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  ssm_rates<LN>(k.in.a, s, p.d, p.sub, p.on, a2);
  if (!LOCAL) ssm_enter<LN, V>(k, s, p, a2, h);
  uint64_t h01 = f2(h[0], h[1]), h23 = f2(h[2], h[3]);
  const uint64_t a01 = f2(a2[0], a2[1]), a23 = f2(a2[2], a2[3]);
  float bias[V], skip[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = k.in.dt_bias != nullptr && p.col_on ? k.in.dt_bias[p.dcol + i] : 0.f;
    skip[i] = !LOCAL && k.in.skip != nullptr && p.col_on ? k.in.skip[p.dcol + i] : 0.f;
  }
  const int t_begin = p.seg * s.seg, t_end = min(s.S, t_begin + s.seg);
  SsmFetch<T, LN, V, false, !LOCAL> f;
  f.load(k.in, nullptr, s, p, t_begin, !LOCAL);
  for (int t0 = t_begin; t0 < t_end; t0 += SSM_TT) {
    Pack<T, V> x[P::ITEMS], z[P::ITEMS];
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      x[i] = f.x[i];
      z[i] = f.z[i];
      const int r = p.row + i * P::ROWS;
      if (r < SSM_TT) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float raw = to_f32(f.dt[i].e[e]) + bias[e];
          const float step = p.col_on && t0 + r < t_end ? (s.softplus ? softplus_f(raw) : raw) : 0.f;   // nothing moves past the end
          s_d[r * CH + p.col + e] = make_float2(step, step * to_f32(x[i].e[e]));
        }
      }
    }
    f.put_bc(s_b, s_c);
    __syncthreads();
    if (t0 + SSM_TT < t_end) f.load(k.in, nullptr, s, p, t0 + SSM_TT, !LOCAL);
    if (!LOCAL && k.ckpt != nullptr && p.on) {
      Pack<float, 4> o;
      unf2(h01, o.e[0], o.e[1]);
      unf2(h23, o.e[2], o.e[3]);
      store_pack<float, 4>(k.ckpt + (((size_t)p.b * s.nt + t0 / SSM_TT) * s.D + p.d) * NP + 4 * p.sub, o);
    }
#pragma unroll
    for (int t = 0; t < SSM_TT; t += TB) {
      float acc[TB];
#pragma unroll
      for (int u = 0; u < TB; ++u) {
        const float2 q = s_d[(t + u) * CH + p.ch];
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(s_b + (t + u) * NP + 4 * p.sub);
        const uint64_t step = f2(q.x, q.x), sx = f2(q.y, q.y);
        float e0, e1, e2, e3;
        unf2(mul2(step, a01), e0, e1);
        unf2(mul2(step, a23), e2, e3);
        h01 = fma2(f2(ex2(e0), ex2(e1)), h01, mul2(sx, b.x));
        h23 = fma2(f2(ex2(e2), ex2(e3)), h23, mul2(sx, b.y));
        if (LOCAL) {
          sum += q.x;
        } else {
          const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(s_c + (t + u) * NP + 4 * p.sub);
          float lo, hi;
          unf2(fma2(c.x, h01, mul2(c.y, h23)), lo, hi);
          acc[u] = lo + hi;
        }
      }
      if (!LOCAL) {
        const float v = lane_sums<LN, TB>(acc, p.sub);
        if (p.sub % (LN / TB) == 0) s_y[(t + p.sub / (LN / TB)) * P::YS + p.ch] = v;
      }
    }
    __syncthreads();
    if (!LOCAL) {
      T* yp = static_cast<T*>(k.y);
#pragma unroll
      for (int i = 0; i < P::ITEMS; ++i) {
        const int r = p.row + i * P::ROWS, t = t0 + r;
        if (!p.col_on || t >= t_end) continue;
        Pack<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float v = fmaf(skip[e], to_f32(x[i].e[e]), s_y[r * P::YS + p.col + e]);
          if (k.in.z != nullptr) {
            const float zz = to_f32(z[i].e[e]);
            v *= zz * logistic_f(zz);
          }
          o.e[e] = from_f32<T>(v);
        }
        store_pack<T, V>(yp + ((size_t)p.b * s.S + t) * s.D + p.dcol, o);
      }
    }
  }
  unf2(h01, h[0], h[1]);
  unf2(h23, h[2], h[3]);
  if (!p.on) return;
  if (LOCAL) {
    const size_t at = ((size_t)p.b * s.nseg + p.seg) * s.D + p.d;
    Pack<float, 4> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.e[i] = h[i];
    store_pack<float, 4>(k.loc_h + at * NP + 4 * p.sub, o);
    if (p.sub == 0) k.loc_sum[at] = sum;
  } else if (k.h_last != nullptr && p.seg == s.nseg - 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * p.sub + i < s.N) k.h_last[((size_t)p.b * s.D + p.d) * s.N + 4 * p.sub + i] = h[i];
  }
}

// One token: bound by the states, in and out once each, 16 bytes a thread (VEC; else element by element).
template <typename T, int LN, bool VEC>
__global__ void __launch_bounds__(SSM_THREADS)
ssm_step_kernel(const T* x, const T* dt, const T* z, const T* b, const T* c, const float* a, const float* skip, const float* dt_bias,
                const float* h, T* y, float* h_new, int B, int D, int N, int G, bool softplus) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int CH = SSM_THREADS / LN;
  const int sub = threadIdx.x % LN;
  const size_t row = (size_t)blockIdx.x * CH + threadIdx.x / LN;   // of (B, D)
  const bool on = row < (size_t)B * D;
  const int d = on ? (int)(row % (unsigned)D) : 0;
  const size_t bi = on ? row / (unsigned)D : 0;
  const size_t bc = (bi * G + d / (D / G)) * N;
  float hv[4], acc = 0.f;
  float step = 0.f, xv = 0.f;
  if (on) {
    const float* hp = h + row * N + 4 * sub;
    const bool any = 4 * sub < N;
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f), r = q;
    if (VEC && any) { q = ld_stream(reinterpret_cast<const float4*>(hp)); r = *reinterpret_cast<const float4*>(a + (size_t)d * N + 4 * sub); }
    float av[4] = {r.x, r.y, r.z, r.w};
    hv[0] = q.x; hv[1] = q.y; hv[2] = q.z; hv[3] = q.w;
    if (!VEC) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = 4 * sub + i < N;
        hv[i] = ok ? hp[i] : 0.f;
        av[i] = ok ? a[(size_t)d * N + 4 * sub + i] : 0.f;
      }
    }
    xv = to_f32(x[row]);
    const float raw = to_f32(dt[row]) + (dt_bias != nullptr ? dt_bias[d] : 0.f);
    step = softplus ? softplus_f(raw) : raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool ok = 4 * sub + i < N;
      const float bv = ok ? to_f32(b[bc + 4 * sub + i]) : 0.f, cv = ok ? to_f32(c[bc + 4 * sub + i]) : 0.f;
      hv[i] = fmaf(ex2(step * (av[i] * kLog2e)), hv[i], step * xv * bv);
      acc = fmaf(cv, hv[i], acc);
    }
    float* op = h_new + row * N + 4 * sub;
    if (VEC) {
      if (any) __stcs(reinterpret_cast<float4*>(op), make_float4(hv[0], hv[1], hv[2], hv[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * sub + i < N) op[i] = hv[i];
    }
  }
#pragma unroll
  for (int o = LN / 2; o >= 1; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (on && sub == 0) {
    float v = skip != nullptr ? fmaf(skip[d], xv, acc) : acc;
    if (z != nullptr) {
      const float zz = to_f32(z[row]);
      v *= zz * logistic_f(zz);
    }
    y[row] = from_f32<T>(v);
  }
}

// ---- launchers ----------------------------------------------------------------------------------------
bool ssm_sizes_ok(int B, int S, int D, int N, int G) {
  if (B <= 0 || S <= 0 || D <= 0 || N <= 0 || N > SSM_MAX_N || G <= 0 || D % G != 0) return false;
  if (S > (1 << 30) || (long long)D * N >= (1ll << 31)) return false;
  const int ch = SSM_THREADS / ssm_lanes(N), Dg = D / G;
  return (long long)B * G * ceil_div(Dg, ch) * 64 < (1ll << 31);
}

// Segments: none while the CTAs of whole sequences give every SM work; two cost as much as they gain (each exponential is then
// taken twice), so at least three.
static int ssm_segments(long long ctas, int nt, int per_sm) {
  const long long room = (long long)per_sm * sm_count();
  long long n = room / ctas;
  if (n > nt / 4) n = nt / 4;      // four tiles each at least
  if (n > 64) n = 64;
  return n < 3 ? 1 : (int)n;
}

SsmDims ssm_dims(int B, int S, int D, int N, int G, bool softplus, const long long* st, bool backward) {
  SsmDims s{};
  s.B = B; s.S = S; s.D = D; s.N = N; s.G = G;
  s.Dg = D / G;
  s.tiles = ceil_div(s.Dg, SSM_THREADS / ssm_lanes(N));
  s.nt = ceil_div(S, SSM_TT);
  const int n = ssm_segments((long long)B * G * s.tiles, s.nt, backward ? 2 : 3);
  s.seg = ceil_div(s.nt, n) * SSM_TT;
  s.nseg = ceil_div(S, s.seg);
  s.softplus = softplus;
  if (st != nullptr) {
    s.xb = st[0]; s.xt = st[1]; s.db = st[2]; s.dt = st[3]; s.zb = st[4]; s.zt = st[5];
    s.bb = st[6]; s.bt = st[7]; s.bg = st[8]; s.cb = st[9]; s.ct = st[10]; s.cg = st[11];
  }
  return s;
}

size_t ssm_ckpt_bytes(int B, int S, int D, int N) { return (size_t)B * ceil_div(S, SSM_TT) * D * 4 * ssm_lanes(N) * sizeof(float); }
size_t ssm_fw_bytes(int B, int S, int D, int N, int G) {
  const SsmDims s = ssm_dims(B, S, D, N, G, false, nullptr, false);
  if (s.nseg == 1) return 0;
  const size_t rows = (size_t)B * s.nseg * D;
  return rows * 4 * ssm_lanes(N) * sizeof(float) + rows * sizeof(float);
}

template <typename T> bool ssm_vec(const SsmIn& in, const SsmDims& s, const void* dy, const void* y) {
  const size_t bytes = sizeof(T) * 4;
  if (s.Dg % 4 != 0) return false;
  const void* p[] = {in.x, in.dt, in.z, dy, y};
  for (const void* q : p)
    if (!fits_access(q, bytes)) return false;
  const long long st[] = {s.xb, s.xt, s.db, s.dt, s.zb, s.zt, s.gb, s.gt};
  for (long long q : st)
    if (!stride_fits(q, sizeof(T), bytes)) return false;
  return true;
}
template bool ssm_vec<float>(const SsmIn&, const SsmDims&, const void*, const void*);
template bool ssm_vec<__nv_bfloat16>(const SsmIn&, const SsmDims&, const void*, const void*);
template bool ssm_vec<__half>(const SsmIn&, const SsmDims&, const void*, const void*);

template <typename T, int LN, int V>
static int ssm_fw_t(const SsmFw& k, const SsmDims& s, cudaStream_t st) {
  const unsigned grid = (unsigned)s.B * s.nseg * s.G * s.tiles;
  const bool overlap = grid <= pdl_max_ctas();
  if (s.nseg > 1)
    if (int rc = launch_pdl(overlap, ssm_fw_kernel<T, LN, V, true>, grid, SSM_THREADS, 0, st, k, s)) return rc;
  return launch_pdl(overlap, ssm_fw_kernel<T, LN, V, false>, grid, SSM_THREADS, 0, st, k, s);
}

int launch_ssm_fw(const SsmIn& in, const long long* strides, void* y, float* h_last, float* ckpt, void* workspace, int B, int S, int D, int N, int G,
                  bool softplus, int dtype, cudaStream_t st) {
  if (!ssm_sizes_ok(B, S, D, N, G)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_SCAN, st);
  const SsmDims s = ssm_dims(B, S, D, N, G, softplus, strides, false);
  const int lanes = ssm_lanes(N);
  SsmFw k{in, y, h_last, ckpt, nullptr, nullptr};
  if (s.nseg > 1) {
    k.loc_h = static_cast<float*>(workspace);
    k.loc_sum = k.loc_h + (size_t)B * s.nseg * D * 4 * lanes;
  }
  MLSTM_DTYPE_SWITCH(dtype, T,
    const bool vec = ssm_vec<T>(in, s, nullptr, y);
    SSM_LANES_SWITCH(lanes, LN, return vec ? ssm_fw_t<T, LN, 4>(k, s, st) : ssm_fw_t<T, LN, 1>(k, s, st);))
  return MLSTM_ERR_DTYPE;
}

int launch_ssm_step(const void* x, const void* dt, const void* z, const void* b, const void* c, const float* a, const float* skip, const float* dt_bias,
                    const float* h, void* y, float* h_new, int B, int D, int N, int G, bool softplus, int dtype, cudaStream_t st) {
  if (!ssm_sizes_ok(B, 1, D, N, G)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_STEP, st);
  const int lanes = ssm_lanes(N);
  const size_t grid = ((size_t)B * D + SSM_THREADS / lanes - 1) / (SSM_THREADS / lanes);
  if (grid >= (1ull << 31)) return MLSTM_ERR_SHAPE;
  const bool vec = N % 4 == 0 && fits_access(a, 16) && fits_access(h, 16) && fits_access(h_new, 16);
#define RUN(LN, VEC)                                                                                                                              \
  return launch_pdl(grid <= pdl_max_ctas(), ssm_step_kernel<T, LN, VEC>, (unsigned)grid, SSM_THREADS, 0, st, (const T*)x, (const T*)dt, (const T*)z, \
                    (const T*)b, (const T*)c, a, skip, dt_bias, h, (T*)y, h_new, B, D, N, G, softplus)
  MLSTM_DTYPE_SWITCH(dtype, T, SSM_LANES_SWITCH(lanes, LN, if (vec) RUN(LN, true); RUN(LN, false);))
#undef RUN
  return MLSTM_ERR_DTYPE;
}

}  // namespace mlstm
