// Selective state space scan, backward.
//
//   dout = dy z sigmoid(z) (or dy);  g_t[n] = dout_t c_t[n] + e_{t+1}[n] g_{t+1}[n],  e_t = exp(step_t a)   (adjoint of the state)
//   dx_t = step_t sum_n g_t b_t + skip dout_t;   dstep_t = x_t sum_n g_t b_t + sum_n a g_t e_t h_{t-1};   ddt = dstep sigmoid(dt + dt_bias)
//   db_t[n] = sum_channels step_t x_t g_t[n];    dc_t[n] = sum_channels dout_t h_t[n];    da[n] = sum_t step_t g_t e_t h_{t-1}
//   dz_t = dy_t (sum_n c_t h_t + skip x_t) sigmoid(z) (1 + z (1 - sigmoid(z)));   dskip = sum_t dout_t x_t;   ddt_bias = sum_t ddt_t
//
// The forward left the state before every tile of 16 tokens; a CTA goes through its tiles from the last to the first, forward
// through the 16 tokens with their states kept in registers, then back.  Bound by instruction issue: some thirty to a state and
// token, two of them exponentials (the second costs less than sixteen more registers would), and the sums over the channels,
// which go through the lanes of a warp (seven shuffles to a token's eight values), the warps of a CTA and, by
// ssm_bw_sums_kernel, the CTAs, each in a fixed order.  Few sequences of few channels are cut into segments as in the forward,
// here from the end: a segment's own adjoint first.
#include "ssm.cuh"

namespace mlstm {

struct SsmBw {
  SsmIn in;
  const void* dy;
  const float* dh_last;     // (B, D, N) or null
  const float* ckpt;        // (B, nt, D, NP)
  void *dx, *ddt, *dz;      // dz null without z
  float* dh0;               // (B, D, N) or null
  float* part_bc;           // (G, tiles, B, S, 2, NP)
  float* part_a;            // (B * nseg, D, NP)
  float* part_d;            // (B * nseg, 2, D): dskip, ddt_bias
  float *loc_g, *loc_sum;   // (B, nseg, D, NP), (B, nseg, D)
};

// The adjoint that enters segment p.seg from behind: e_{t+1} g_{t+1} at its last token
template <int LN, int V>
__device__ __forceinline__ void ssm_enter_back(const SsmBw& k, const SsmDims& s, const SsmPlace<LN, V>& p, const float (&a2)[4], float (&r)[4]) {
  constexpr int NP = 4 * LN;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = k.dh_last != nullptr && p.on && 4 * p.sub + i < s.N ? k.dh_last[((size_t)p.b * s.D + p.d) * s.N + 4 * p.sub + i] : 0.f;
  if (!p.on) return;
  for (int j = s.nseg - 1; j > p.seg; --j) {
    const size_t at = ((size_t)p.b * s.nseg + j) * s.D + p.d;
    const float sum = k.loc_sum[at];
    const Pack<float, 4> l = load_pack<float, 4>(k.loc_g + at * NP + 4 * p.sub);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fmaf(ex2(sum * a2[i]), r[i], l.e[i]);
  }
}

__device__ __forceinline__ float gate_f(float z) { return z * logistic_f(z); }

// A segment's own adjoint (nothing entering from behind) as it leaves at its first token, and the sum of its steps.
template <typename T, int LN, int V>
__global__ void __launch_bounds__(SSM_THREADS, 3)
ssm_bw_local_kernel(SsmBw k, SsmDims s) {
  using P = SsmPlace<LN, V>;
  constexpr int CH = P::CH, NP = P::NP;
  __shared__ float2 s_d[SSM_TT * CH];                  // (step, dout)
  __shared__ __align__(16) float s_c[SSM_TT * NP];
  pdl_launch_dependents();
  pdl_wait();
  const P p(s);
  float a2[4], r[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f, bias[V];
  ssm_rates<LN>(k.in.a, s, p.d, p.sub, p.on, a2);
#pragma unroll
  for (int i = 0; i < V; ++i) bias[i] = k.in.dt_bias != nullptr && p.col_on ? k.in.dt_bias[p.dcol + i] : 0.f;
  const int t_begin = p.seg * s.seg, t_end = min(s.S, t_begin + s.seg);
  SsmIn in = k.in;
  in.b = in.c;   // of the two only c is needed
  SsmDims sc = s;
  sc.bb = s.cb; sc.bt = s.ct; sc.bg = s.cg;
  SsmFetch<T, LN, V, true, false> f;
  const int t_last = t_begin + (t_end - 1 - t_begin) / SSM_TT * SSM_TT;
  f.load(in, k.dy, sc, p, t_last, true);
  for (int t0 = t_last; t0 >= t_begin; t0 -= SSM_TT) {
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      const int q = p.row + i * P::ROWS;
      if (q < SSM_TT) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float raw = to_f32(f.dt[i].e[e]) + bias[e];
          const float step = p.col_on && t0 + q < t_end ? (s.softplus ? softplus_f(raw) : raw) : 0.f;
          const float dy = to_f32(f.dy[i].e[e]);
          s_d[q * CH + p.col + e] = make_float2(step, in.z != nullptr ? dy * gate_f(to_f32(f.z[i].e[e])) : dy);
        }
      }
    }
    f.put_bc(s_c, nullptr);
    __syncthreads();
    if (t0 > t_begin) f.load(in, k.dy, sc, p, t0 - SSM_TT, true);
#pragma unroll 4
    for (int t = SSM_TT - 1; t >= 0; --t) {
      const float2 q = s_d[t * CH + p.ch];
      const float4 c = *reinterpret_cast<const float4*>(s_c + t * NP + 4 * p.sub);
      r[0] = ex2(q.x * a2[0]) * fmaf(q.y, c.x, r[0]);
      r[1] = ex2(q.x * a2[1]) * fmaf(q.y, c.y, r[1]);
      r[2] = ex2(q.x * a2[2]) * fmaf(q.y, c.z, r[2]);
      r[3] = ex2(q.x * a2[3]) * fmaf(q.y, c.w, r[3]);
      sum += q.x;
    }
    __syncthreads();
  }
  if (!p.on) return;
  const size_t at = ((size_t)p.b * s.nseg + p.seg) * s.D + p.d;
  Pack<float, 4> o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.e[i] = r[i];
  store_pack<float, 4>(k.loc_g + at * NP + 4 * p.sub, o);
  if (p.sub == 0) k.loc_sum[at] = sum;
}

// Shared memory of the backward, in floats
template <int LN, int V> struct SsmBwSmem {
  using P = SsmPlace<LN, V>;
  static constexpr int TF = LN <= 4 ? SSM_TT : 64 / LN;          // tokens whose channel sums wait for the other warps
  static constexpr int D4 = 0, B = D4 + 4 * SSM_TT * P::CH, C = B + SSM_TT * P::NP, S1 = C + SSM_TT * P::NP, S2 = S1 + SSM_TT * P::YS,
                       YP = S2 + SSM_TT * P::YS, PART = YP + SSM_TT * P::YS, END = PART + 8 * TF * 2 * P::NP;
  static constexpr size_t BYTES = END * sizeof(float);
};

template <typename T, int LN, int V>
__global__ void __launch_bounds__(SSM_THREADS, 2)
ssm_bw_kernel(SsmBw k, SsmDims s) {
  using P = SsmPlace<LN, V>;
  using M = SsmBwSmem<LN, V>;
  constexpr int CH = P::CH, NP = P::NP, TB = LN < 8 ? LN : 8, REP = LN / TB, TF = M::TF, LC = P::LC;
  extern __shared__ __align__(16) float sm[];
  float4* s_d = reinterpret_cast<float4*>(sm + M::D4);           // (step, step x, dout, -)
  float *s_b = sm + M::B, *s_c = sm + M::C, *s_s1 = sm + M::S1, *s_s2 = sm + M::S2, *s_yp = sm + M::YP, *s_part = sm + M::PART;
  pdl_launch_dependents();
  pdl_wait();
  const P p(s);
  const bool gate = k.in.z != nullptr;
  float a2[4], r[4], da[4] = {0.f, 0.f, 0.f, 0.f};
  ssm_rates<LN>(k.in.a, s, p.d, p.sub, p.on, a2);
  ssm_enter_back<LN, V>(k, s, p, a2, r);
  float bias[V], skip[V], dskip[V], dbias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = k.in.dt_bias != nullptr && p.col_on ? k.in.dt_bias[p.dcol + i] : 0.f;
    skip[i] = k.in.skip != nullptr && p.col_on ? k.in.skip[p.dcol + i] : 0.f;
    dskip[i] = dbias[i] = 0.f;
  }
  const int t_begin = p.seg * s.seg, t_end = min(s.S, t_begin + s.seg);
  const int t_last = t_begin + (t_end - 1 - t_begin) / SSM_TT * SSM_TT;
  SsmFetch<T, LN, V, true, true> f;
  f.load(k.in, k.dy, s, p, t_last, true);
  float* bc = k.part_bc + ((size_t)(p.g * s.tiles + p.tile) * s.B + p.b) * s.S * (2 * NP);
  const float* ck = k.ckpt + ((size_t)p.b * s.nt * s.D + (p.on ? p.d : 0)) * NP + 4 * p.sub;
  Pack<float, 4> h0 = zero_pack<float, 4>();
  if (p.on) h0 = load_pack<float, 4>(ck + (size_t)(t_last / SSM_TT) * s.D * NP);
  for (int t0 = t_last; t0 >= t_begin; t0 -= SSM_TT) {
    Pack<T, V> x[P::ITEMS], z[P::ITEMS], dy[P::ITEMS], dt[P::ITEMS];
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      x[i] = f.x[i]; z[i] = f.z[i]; dy[i] = f.dy[i]; dt[i] = f.dt[i];
      const int q = p.row + i * P::ROWS;
      if (q < SSM_TT) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float raw = to_f32(dt[i].e[e]) + bias[e];
          const float step = p.col_on && t0 + q < t_end ? (s.softplus ? softplus_f(raw) : raw) : 0.f;
          const float g = to_f32(dy[i].e[e]);
          s_d[q * CH + p.col + e] = make_float4(step, step * to_f32(x[i].e[e]), gate ? g * gate_f(to_f32(z[i].e[e])) : g, 0.f);
        }
      }
    }
    f.put_bc(s_b, s_c);
    __syncthreads();
    float h[SSM_TT][4];
    float hb[4] = {h0.e[0], h0.e[1], h0.e[2], h0.e[3]};   // before the tile
    if (t0 > t_begin) {
      f.load(k.in, k.dy, s, p, t0 - SSM_TT, true);
      if (p.on) h0 = load_pack<float, 4>(ck + (size_t)(t0 / SSM_TT - 1) * s.D * NP);
    }
#pragma unroll
    for (int t = 0; t < SSM_TT; t += TB) {
      float acc[TB];
#pragma unroll
      for (int u = 0; u < TB; ++u) {
        const float4 q = s_d[(t + u) * CH + p.ch];
        const float4 b = *reinterpret_cast<const float4*>(s_b + (t + u) * NP + 4 * p.sub);
        const float bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) h[t + u][i] = fmaf(ex2(q.x * a2[i]), t + u == 0 ? hb[i] : h[t + u == 0 ? 0 : t + u - 1][i], q.y * bv[i]);
        if (gate) {
          const float4 c = *reinterpret_cast<const float4*>(s_c + (t + u) * NP + 4 * p.sub);
          acc[u] = fmaf(c.x, h[t + u][0], fmaf(c.y, h[t + u][1], fmaf(c.z, h[t + u][2], c.w * h[t + u][3])));
        }
      }
      if (gate) {
        const float v = lane_sums<LN, TB>(acc, p.sub);
        if (p.sub % REP == 0) s_yp[(t + p.sub / REP) * P::YS + p.ch] = v;
      }
    }
#pragma unroll
    for (int tb = SSM_TT - TB; tb >= 0; tb -= TB) {
      float acc1[TB], acc2[TB];
#pragma unroll
      for (int u = TB - 1; u >= 0; --u) {
        const int t = tb + u;
        const float4 q = s_d[t * CH + p.ch];
        const float4 b = *reinterpret_cast<const float4*>(s_b + t * NP + 4 * p.sub);
        const float4 c = *reinterpret_cast<const float4*>(s_c + t * NP + 4 * p.sub);
        const float bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
        float v[8];
        acc1[u] = acc2[u] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = fmaf(q.z, cv[i], r[i]);
          acc1[u] = fmaf(g, bv[i], acc1[u]);
          r[i] = ex2(q.x * a2[i]) * g;
          const float w = r[i] * (t == 0 ? hb[i] : h[t == 0 ? 0 : t - 1][i]);
          acc2[u] = fmaf(a2[i], w, acc2[u]);
          da[i] = fmaf(q.x, w, da[i]);
          v[i] = q.y * g;
          v[4 + i] = q.z * h[t][i];
        }
        // over the channels of the warp: each step halves the values that a lane still carries
        int first = 0;
#pragma unroll
        for (int bit = LC / 2, n = 8; bit >= 1; bit >>= 1) {
          if (n > 1) {
            n >>= 1;
            const bool up = (p.chl & bit) != 0;
#pragma unroll
            for (int j = 0; j < n; ++j) {
              const float mine = up ? v[j + n] : v[j], theirs = up ? v[j] : v[j + n];
              v[j] = mine + __shfl_xor_sync(0xffffffffu, theirs, bit * LN);
            }
            first += up ? n : 0;
          } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit * LN);
          }
        }
        constexpr int LEFT = LC >= 8 ? 1 : 8 / LC;
        if (LC <= 8 || p.chl % (LC > 8 ? LC / 8 : 1) == 0) {
#pragma unroll
          for (int j = 0; j < LEFT; ++j) {
            const int e = first + j;
            s_part[((p.warp * TF + t % TF) * 2 + e / 4) * NP + 4 * p.sub + e % 4] = v[j];
          }
        }
        if (t % TF == 0) {   // TF tokens are there: over the warps
          __syncthreads();
          for (int e = threadIdx.x; e < TF * 2 * NP; e += SSM_THREADS) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) a += s_part[w * TF * 2 * NP + e];
            const int tt = t0 + t + e / (2 * NP);
            if (tt < t_end) bc[(size_t)tt * (2 * NP) + e % (2 * NP)] = a;
          }
          if (t > 0) __syncthreads();
        }
      }
      const float v1 = lane_sums<LN, TB>(acc1, p.sub), v2 = lane_sums<LN, TB>(acc2, p.sub);
      if (p.sub % REP == 0) {
        s_s1[(tb + p.sub / REP) * P::YS + p.ch] = v1;
        s_s2[(tb + p.sub / REP) * P::YS + p.ch] = v2;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      const int q = p.row + i * P::ROWS, t = t0 + q;
      if (!p.col_on || t >= t_end) continue;
      Pack<T, V> ox, ot, oz;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float4 d4 = s_d[q * CH + p.col + e];
        const float s1 = s_s1[q * P::YS + p.col + e], s2 = s_s2[q * P::YS + p.col + e] * kLn2;
        const float xv = to_f32(x[i].e[e]);
        ox.e[e] = from_f32<T>(fmaf(d4.x, s1, skip[e] * d4.z));
        float ddt = fmaf(xv, s1, s2);
        if (s.softplus) ddt *= logistic_f(to_f32(dt[i].e[e]) + bias[e]);
        ot.e[e] = from_f32<T>(ddt);
        dbias[e] += ddt;
        dskip[e] = fmaf(d4.z, xv, dskip[e]);
        if (gate) {
          const float zz = to_f32(z[i].e[e]), sg = logistic_f(zz);
          oz.e[e] = from_f32<T>(to_f32(dy[i].e[e]) * fmaf(skip[e], xv, s_yp[q * P::YS + p.col + e]) * sg * fmaf(zz, 1.f - sg, 1.f));
        }
      }
      const size_t at = ((size_t)p.b * s.S + t) * s.D + p.dcol;
      store_pack<T, V>(static_cast<T*>(k.dx) + at, ox);
      store_pack<T, V>(static_cast<T*>(k.ddt) + at, ot);
      if (gate) store_pack<T, V>(static_cast<T*>(k.dz) + at, oz);
    }
    __syncthreads();   // the tile's arrays are free
  }
  const size_t row = (size_t)p.b * s.nseg + p.seg;
  if (p.on) {
    Pack<float, 4> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.e[i] = da[i];
    store_pack<float, 4>(k.part_a + (row * s.D + p.d) * NP + 4 * p.sub, o);
    if (k.dh0 != nullptr && p.seg == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * p.sub + i < s.N) k.dh0[((size_t)p.b * s.D + p.d) * s.N + 4 * p.sub + i] = r[i];
    }
  }
  // dskip and ddt_bias: over the threads that share a channel
  float* s_x = sm;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (p.row < SSM_TT) {
#pragma unroll
      for (int e = 0; e < V; ++e) s_x[p.row * CH + p.col + e] = which == 0 ? dskip[e] : dbias[e];
    }
    __syncthreads();
    constexpr int N_ROWS = P::ROWS < SSM_TT ? P::ROWS : SSM_TT;
    for (int c = threadIdx.x; c < CH; c += SSM_THREADS) {
      float a = 0.f;
#pragma unroll
      for (int q = 0; q < N_ROWS; ++q) a += s_x[q * CH + c];
      if (p.tile * CH + c < s.Dg) k.part_d[(row * 2 + which) * s.D + p.g * s.Dg + p.tile * CH + c] = a;
    }
    __syncthreads();
  }
}

// The sums over CTAs, in their order: db and dc over the channel tiles, da, dskip and ddt_bias over sequences and segments.
struct SsmSums {
  const float *part_bc, *part_a, *part_d;
  void *db, *dc;                       // (B, S, G, N)
  float *da, *dskip, *ddt_bias;        // dskip, ddt_bias may be null
  int NP;
  size_t n_bc, n_a;                    // threads of each kind; n_bc: 2 * B * S * G * NP
};
template <typename T>
__global__ void __launch_bounds__(256)
ssm_bw_sums_kernel(SsmSums q, SsmDims s) {
  pdl_launch_dependents();
  pdl_wait();
  size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id < q.n_bc) {
    const int n = (int)(id % q.NP);
    size_t k = id / q.NP;
    const int which = (int)(k % 2);
    k /= 2;
    const size_t per_tile = (size_t)s.B * s.S;
    const size_t tok = k % per_tile;
    const int g = (int)(k / per_tile);
    if (n >= s.N) return;
    const float* src = q.part_bc + ((size_t)g * s.tiles * per_tile + tok) * 2 * q.NP + which * q.NP + n;
    float a = 0.f;
    for (int t = 0; t < s.tiles; ++t) a += src[t * per_tile * 2 * q.NP];
    static_cast<T*>(which == 0 ? q.db : q.dc)[(tok * s.G + g) * s.N + n] = from_f32<T>(a);
    return;
  }
  id -= q.n_bc;
  const int rows = s.B * s.nseg;
  if (id < q.n_a) {
    const int n = (int)(id % q.NP);
    const size_t d = id / q.NP;
    if (n >= s.N) return;
    float a = 0.f;
    for (int t = 0; t < rows; ++t) a += q.part_a[((size_t)t * s.D + d) * q.NP + n];
    q.da[d * s.N + n] = a;
    return;
  }
  id -= q.n_a;
  if (id >= 2 * (size_t)s.D) return;
  const int which = id >= (size_t)s.D;
  const size_t d = id - (which ? s.D : 0);
  float* out = which ? q.ddt_bias : q.dskip;
  if (out == nullptr) return;
  float a = 0.f;
  for (int t = 0; t < rows; ++t) a += q.part_d[((size_t)t * 2 + which) * s.D + d];
  out[d] = a;
}

// ---- launchers ----------------------------------------------------------------------------------------
SsmDims ssm_dims(int B, int S, int D, int N, int G, bool softplus, const long long* strides, bool backward);
template <typename T> bool ssm_vec(const SsmIn& in, const SsmDims& s, const void* dy, const void* y);

struct SsmBwLayout { size_t bc, a, d, g, sum, end; };
static SsmBwLayout ssm_bw_layout(const SsmDims& s) {
  const size_t np = 4 * ssm_lanes(s.N), rows = (size_t)s.B * s.nseg;
  SsmBwLayout l{};
  l.bc = 0;
  l.a = align_up(l.bc + (size_t)s.G * s.tiles * s.B * s.S * 2 * np * sizeof(float), 256);
  l.d = align_up(l.a + rows * s.D * np * sizeof(float), 256);
  l.g = align_up(l.d + rows * 2 * s.D * sizeof(float), 256);
  l.sum = align_up(l.g + (s.nseg > 1 ? rows * s.D * np * sizeof(float) : 0), 256);
  l.end = align_up(l.sum + (s.nseg > 1 ? rows * s.D * sizeof(float) : 0), 256);
  return l;
}
size_t ssm_bw_bytes(int B, int S, int D, int N, int G) { return ssm_bw_layout(ssm_dims(B, S, D, N, G, false, nullptr, true)).end; }

template <typename T, int LN, int V>
static int ssm_bw_t(const SsmBw& k, const SsmDims& s, cudaStream_t st) {
  const unsigned grid = (unsigned)s.B * s.nseg * s.G * s.tiles;
  const bool overlap = grid <= pdl_max_ctas();
  if (s.nseg > 1)
    if (int rc = launch_pdl(overlap, ssm_bw_local_kernel<T, LN, V>, grid, SSM_THREADS, 0, st, k, s)) return rc;
  constexpr size_t smem = SsmBwSmem<LN, V>::BYTES;
  auto kern = ssm_bw_kernel<T, LN, V>;
  if (smem > 48 * 1024) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_pdl(overlap, kern, grid, SSM_THREADS, smem, st, k, s);
}

int launch_ssm_bw(const SsmIn& in, const long long* strides, const void* dy, const long long* gs, const float* dh_last, const float* ckpt, void* dx,
                  void* ddt, void* dz, void* db, void* dc, float* da, float* dskip, float* ddt_bias, float* dh0, void* workspace, int B, int S, int D,
                  int N, int G, bool softplus, int dtype, cudaStream_t st) {
  if (!ssm_sizes_ok(B, S, D, N, G)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_SCAN, st);
  SsmDims s = ssm_dims(B, S, D, N, G, softplus, strides, true);
  s.gb = gs[0]; s.gt = gs[1];
  const int lanes = ssm_lanes(N), np = 4 * lanes;
  const SsmBwLayout l = ssm_bw_layout(s);
  char* w = static_cast<char*>(workspace);
  auto at = [&](size_t o) { return reinterpret_cast<float*>(w + o); };
  const SsmBw k{in, dy, dh_last, ckpt, dx, ddt, dz, dh0, at(l.bc), at(l.a), at(l.d), at(l.g), at(l.sum)};
  SsmSums q{k.part_bc, k.part_a, k.part_d, db, dc, da, dskip, ddt_bias, np, (size_t)2 * B * S * G * np, (size_t)D * np};
  const size_t threads = q.n_bc + q.n_a + 2 * (size_t)D, grid = (threads + 255) / 256;
  if (grid >= (1ull << 31)) return MLSTM_ERR_SHAPE;
  int rc = MLSTM_ERR_DTYPE;
  MLSTM_DTYPE_SWITCH(dtype, T,
    const bool vec = ssm_vec<T>(in, s, dy, dx) && ssm_vec<T>(in, s, ddt, dz);
    SSM_LANES_SWITCH(lanes, LN, rc = vec ? ssm_bw_t<T, LN, 4>(k, s, st) : ssm_bw_t<T, LN, 1>(k, s, st);)
    if (rc == MLSTM_OK) rc = launch_pdl(grid <= pdl_max_ctas(), ssm_bw_sums_kernel<T>, (unsigned)grid, 256, 0, st, q, s);)
  return rc;
}

}  // namespace mlstm
