// Selective state space scan, backward.
//
//   dout = dy z sigmoid(z) (or dy);  g_t[n] = dout_t c_t[n] + e_{t+1}[n] g_{t+1}[n],  e_t = exp(step_t a)   (adjoint of the state)
//   dx_t = step_t sum_n g_t b_t + skip dout_t;   dstep_t = x_t sum_n g_t b_t + sum_n a g_t e_t h_{t-1};   ddt = dstep sigmoid(dt + dt_bias)
//   db_t[n] = sum_channels step_t x_t g_t[n];    dc_t[n] = sum_channels dout_t h_t[n];    da[n] = sum_t step_t g_t e_t h_{t-1}
//   dz_t = dy_t (sum_n c_t h_t + skip x_t) sigmoid(z) (1 + z (1 - sigmoid(z)));   dskip = sum_t dout_t x_t;   ddt_bias = sum_t ddt_t
//
// The forward left the state before every tile of 16 tokens; a CTA goes through its tiles from the last to the first, eight tokens at a
// time: forward with their states kept in registers, then back (for a tile's second half first through its first half without
// keeping any: 2.5 exponentials a state and token; all sixteen tokens' states do not fit the registers of four CTAs to an SM).  Shared
// memory holds fewer than four with up to 8 states (two, one in f32) and, in f32, with 9 to 16 and 65 to 128 (three).  The
// sums over the channels go through the lanes of a warp (seven shuffles to a token's eight values, of two channels at once), the
// warps of a CTA and, by ssm_bw_sums_kernel, the CTAs, each in a fixed order.  Few sequences of few channels are cut into segments
// as in the forward, here from the end: a segment's own adjoint first (bound by the special function units, 80 % busy).
// 4 x 2048 x 2048 channels of 16 states in bf16, nine segments: 540 us; alone, with cold caches, own adjoints 93, backward 444, sums 20.
// The backward issues 30 instructions to a state and token: its schedulers are 56 % busy, shared memory 58 %, special functions 44 %,
// with 3.5 warps to a scheduler, and its 128 registers spill 228 bytes a thread; one channel to a thread (twice the warps, 15 % more
// instructions) and two to four CTAs to an SM took the same time.
#include <algorithm>

#include "ssm.cuh"

namespace mlstm {

constexpr int SSM_BW_C = 2, SSM_BW_LOCAL_C = 2;   // channels to a thread

struct SsmBw {
  SsmIn in;
  const void* dy;
  const float* dh_last;     // (B, D, N) or null
  const float* ckpt;        // (B, nt, D, NP)
  void *dx, *ddt, *dz;      // dz null without z
  float* dh0;               // (B, D, N) or null
  float* part_bc;           // (G, parts, rows, seg, 2, NP)
  float* part_a;            // (B * nseg, D, NP)
  float* part_d;            // (B * nseg, 2, D): dskip, ddt_bias
  float *loc_g, *loc_sum;   // (B, nseg, D, NP), (B, nseg, D)
};

// Shared memory of a segment's own adjoint, in bytes
template <typename T, int LN, int V> struct SsmBwLocalSmem {
  using P = SsmPlace<LN, V, SSM_BW_LOCAL_C>;
  using Ring = SsmRing<T, P, V, 3, 1>;
  static constexpr size_t D = 0, C = D + sizeof(float2) * SSM_TT * P::CH, X = C + sizeof(float) * SSM_TT * P::NP, BYTES = X + Ring::BYTES;
  static constexpr int RESIDENT = scan_resident(BYTES, 5);
};

// A segment's own adjoint (nothing entering from behind) as it leaves at its first token, and the sum of its steps.
template <typename T, int LN, int V>
__global__ void __launch_bounds__(SsmBwLocalSmem<T, LN, V>::P::THREADS, SsmBwLocalSmem<T, LN, V>::RESIDENT)
ssm_bw_local_kernel(SsmBw k, SsmDims s, int nseg) {
  using M = SsmBwLocalSmem<T, LN, V>;
  using P = typename M::P;
  using Ring = typename M::Ring;
  constexpr int CH = P::CH, NP = P::NP, AHEAD = Ring::STAGES - 1;
  extern __shared__ __align__(16) char sm[];
  float2* s_d = reinterpret_cast<float2*>(sm + M::D);  // (step, dout)
  float* s_c = reinterpret_cast<float*>(sm + M::C);
  const Ring ring{reinterpret_cast<T*>(sm + M::X)};    // dt, z, dy; c
  pdl_launch_dependents();
  pdl_wait();
  const P p(s, nseg, 1);
  uint64_t a2[P::C][2], r[P::C][2];
  float bias[V], sum[P::C];
#pragma unroll
  for (int c = 0; c < P::C; ++c) { r[c][0] = r[c][1] = 0ull; sum[c] = 0.f; }
  ssm_rates(k.in.a, s, p, a2);
#pragma unroll
  for (int i = 0; i < V; ++i) bias[i] = k.in.dt_bias != nullptr && p.col_on ? k.in.dt_bias[p.dcol + i] : 0.f;
  const int t_begin = p.seg * s.seg, t_end = min(s.S, t_begin + s.seg);
  const int t_last = t_begin + (t_end - 1 - t_begin) / SSM_TT * SSM_TT;
  const bool gate = k.in.z != nullptr;
  const SsmSource from_dt = ssm_source<T>(k.in.dt, p.b * s.db + p.dcol, s.dt), from_z = ssm_source<T>(k.in.z, p.b * s.zb + p.dcol, s.zt),
                  from_dy = ssm_source<T>(k.dy, p.b * s.gb + p.dcol, s.gt), from_c = Ring::source_bc(k.in.c, p, s.cb, s.ct, s.cg);
  auto fetch = [&](int t0) {
    if (t0 >= t_begin) {
      ring.copy(s, p, t0, 0, from_dt);
      if (gate) ring.copy(s, p, t0, 1, from_z);
      ring.copy(s, p, t0, 2, from_dy);
      ring.copy_bc(s, p, t0, 0, from_c);
    }
    cp_commit();
  };
  ring.clear(s, p);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(t_last - i * SSM_TT);
  for (int t0 = t_last; t0 >= t_begin; t0 -= SSM_TT) {
    const int tile = t0 / SSM_TT;
    cp_wait<AHEAD - 1>();
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      const int q = p.row + i * P::ROWS;
      if (q >= SSM_TT) continue;
      float dt[V], step[V], g[V];
      ring.get(tile, 0, i, p, dt);
      ring.get(tile, 2, i, p, g);
      ssm_step_v<T, V>(dt, bias, s.softplus, t0 + q >= t_end, step);
      if (gate) {
        float zv[V], sg[V];
        ring.get(tile, 1, i, p, zv);
        logistic_v<T, V>(zv, sg);
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] *= zv[e] * sg[e];
      }
      Pack<float2, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.e[e] = make_float2(step[e], g[e]);
      store_pack<float2, V>(s_d + q * CH + p.col, o);
    }
    ring.put(tile, 0, s_c);
    __syncthreads();
    fetch(t0 - AHEAD * SSM_TT);
#pragma unroll 4
    for (int t = SSM_TT - 1; t >= 0; --t) {
      const Pack<float2, P::C> q = load_pack<float2, P::C>(s_d + t * CH + p.ch);
      const ulonglong2 c2 = *reinterpret_cast<const ulonglong2*>(s_c + t * NP + 4 * p.sub);
#pragma unroll
      for (int c = 0; c < P::C; ++c) {
        const uint64_t step = f2(q.e[c].x, q.e[c].x), g = f2(q.e[c].y, q.e[c].y);
        r[c][0] = mul2(ex2_pair(mul2(step, a2[c][0])), fma2(g, c2.x, r[c][0]));
        r[c][1] = mul2(ex2_pair(mul2(step, a2[c][1])), fma2(g, c2.y, r[c][1]));
        sum[c] += q.e[c].x;
      }
    }
    __syncthreads();
  }
  const size_t at = ((size_t)p.b * s.nseg + p.seg) * s.D + p.d;
  ssm_put_states(k.loc_g, p, at, r);
#pragma unroll
  for (int c = 0; c < P::C; ++c)
    if (p.on[c] && p.sub == 0) k.loc_sum[at + c] = sum[c];
}

// Shared memory of the backward, in bytes
template <typename T, int LN, int V> struct SsmBwSmem {
  using P = SsmPlace<LN, V, SSM_BW_C>;
  static constexpr int TF = LN <= 8 ? SSM_TT / 2 : 64 / LN;          // tokens whose channel sums wait for the other warps
  using Ring = SsmRing<T, P, V, 4, 2>;
  static constexpr size_t Q = 0, G = Q + sizeof(float2) * SSM_TT * P::CH, B = G + sizeof(float) * SSM_TT * P::CH, C = B + sizeof(float) * SSM_TT * P::NP,
                          SUMS = C + sizeof(float) * SSM_TT * P::NP, PART = SUMS + sizeof(float) * (3 * SSM_TT * P::YS + 16),
                          X = PART + sizeof(float) * P::WARPS * TF * 2 * P::NP, BYTES = X + Ring::BYTES;
  static constexpr int RESIDENT = scan_resident(BYTES, 4);
};

// One tile of channels of a segment.  first: the sums over its channels begin the CTA's part of db and dc, else they are added.
template <typename T, int LN, int V>
__device__ __forceinline__ void ssm_bw_tile(const SsmBw& k, const SsmDims& s, const typename SsmBwSmem<T, LN, V>::P& p, bool first_turn, char* sm) {
  using M = SsmBwSmem<T, LN, V>;
  using P = typename M::P;
  using Ring = typename M::Ring;
  using Sums = LaneSums<LN>;
  constexpr int CH = P::CH, NP = P::NP, TF = M::TF, LC = P::LC, HALF = SSM_TT / 2, AHEAD = Ring::STAGES - 1;
  float2* s_q = reinterpret_cast<float2*>(sm + M::Q);            // (step, step x)
  float *s_g = reinterpret_cast<float*>(sm + M::G), *s_b = reinterpret_cast<float*>(sm + M::B), *s_c = reinterpret_cast<float*>(sm + M::C);
  float *s_sum = reinterpret_cast<float*>(sm + M::SUMS), *s_part = reinterpret_cast<float*>(sm + M::PART);
  constexpr int S2 = SSM_TT * P::YS + 16;                        // (the two sums of a warp in different banks)
  float* s_yp = s_sum + S2 + SSM_TT * P::YS;                     // s_sum: sum g b and, from S2 on, sum a g e h; s_yp: sum c h
  const Ring ring{reinterpret_cast<T*>(sm + M::X)};              // x, dt, z, dy; b, c
  const bool gate = k.in.z != nullptr;
  uint64_t a2[P::C][2], r[P::C][2], da[P::C][2];
#pragma unroll
  for (int c = 0; c < P::C; ++c) da[c][0] = da[c][1] = 0ull;
  ssm_rates(k.in.a, s, p, a2);
  ssm_load_states(k.dh_last, s, p, (size_t)p.b * s.D + p.d, r);
  ssm_fold<true>(k.loc_g, k.loc_sum, p.seg + 1, s.nseg, s, p, a2, r);
  float dskip[V], dbias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) dskip[i] = dbias[i] = 0.f;
  const int t_begin = p.seg * s.seg, t_end = min(s.S, t_begin + s.seg);
  const int t_last = t_begin + (t_end - 1 - t_begin) / SSM_TT * SSM_TT;
  auto fetch = [&](int t0) {   // (the sources anew each time: the loop has no registers left for them)
    if (t0 >= t_begin) {
      ring.copy(s, p, t0, 0, ssm_source<T>(k.in.x, p.b * s.xb + p.dcol, s.xt));
      ring.copy(s, p, t0, 1, ssm_source<T>(k.in.dt, p.b * s.db + p.dcol, s.dt));
      if (gate) ring.copy(s, p, t0, 2, ssm_source<T>(k.in.z, p.b * s.zb + p.dcol, s.zt));
      ring.copy(s, p, t0, 3, ssm_source<T>(k.dy, p.b * s.gb + p.dcol, s.gt));
      ring.copy_bc(s, p, t0, 0, Ring::source_bc(k.in.b, p, s.bb, s.bt, s.bg));
      ring.copy_bc(s, p, t0, 1, Ring::source_bc(k.in.c, p, s.cb, s.ct, s.cg));
    }
    cp_commit();
  };
  ring.clear(s, p);
  auto param = [&](const float* v, float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = v != nullptr && p.col_on ? v[p.dcol + i] : 0.f;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(t_last - i * SSM_TT);
  // (of token t_begin on)
  float* bc = k.part_bc + ((size_t)(p.g * s.parts + p.tile / s.per_cta) * s.rows + (p.b * s.nseg + p.seg - s.row0)) * s.seg * (2 * NP);
  for (int t0 = t_last; t0 >= t_begin; t0 -= SSM_TT) {
    const int tile = t0 / SSM_TT;
    cp_wait<AHEAD - 1>();
    {
      float bias[V];
      param(k.in.dt_bias, bias);
#pragma unroll
      for (int i = 0; i < P::ITEMS; ++i) {
        const int q = p.row + i * P::ROWS, at = q * CH + p.col;
        if (q >= SSM_TT) continue;
        float xv[V], dt[V], step[V], g[V];
        ring.get(tile, 0, i, p, xv);
        ring.get(tile, 1, i, p, dt);
        ring.get(tile, 3, i, p, g);
        ssm_step_v<T, V>(dt, bias, s.softplus, t0 + q >= t_end, step);
        Pack<float2, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.e[e] = make_float2(step[e], step[e] * xv[e]);
        store_pack<float2, V>(s_q + at, o);
        if (gate) {
          float zv[V], sg[V];
          ring.get(tile, 2, i, p, zv);
          logistic_v<T, V>(zv, sg);
#pragma unroll
          for (int e = 0; e < V; ++e) g[e] *= zv[e] * sg[e];
        }
        store_pack<float, V>(s_g + at, pack<float, V>(g));
      }
    }
    ring.put(tile, 0, s_b);
    ring.put(tile, 1, s_c);
    __syncthreads();
    fetch(t0 - AHEAD * SSM_TT);
    // one token onwards
    auto onward = [&](int t, const uint64_t (&from)[P::C][2], uint64_t (&to)[P::C][2]) {
      const Pack<float2, P::C> q = load_pack<float2, P::C>(s_q + t * CH + p.ch);
      const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(s_b + t * NP + 4 * p.sub);
#pragma unroll
      for (int c = 0; c < P::C; ++c) {
        const uint64_t step = f2(q.e[c].x, q.e[c].x), sx = f2(q.e[c].y, q.e[c].y);
        to[c][0] = fma2(ex2_pair(mul2(step, a2[c][0])), from[c][0], mul2(sx, b.x));
        to[c][1] = fma2(ex2_pair(mul2(step, a2[c][1])), from[c][1], mul2(sx, b.y));
      }
    };
    // The states of eight tokens are kept at a time: for the tile's second half first through the first without keeping any.
    const bool full = t0 + HALF < t_end;
#pragma unroll 1
    for (int half = full ? HALF : 0; half >= 0; half -= HALF) {
      uint64_t h[HALF + 1][P::C][2];
      ssm_get_states(k.ckpt, p, ((size_t)p.b * s.nt + t0 / SSM_TT) * s.D + p.d, h[0]);   // (fetched when it is needed: the tile's work hides it)
#pragma unroll 4
      for (int t = 0; t < half; ++t) onward(t, h[0], h[0]);
      constexpr int UF = 4 / P::C, UB = 2 / P::C;   // tokens whose sums over the states are taken together
#pragma unroll
      for (int t = 0; t < HALF; t += UF) {
        float acc[4];
#pragma unroll
        for (int u = 0; u < UF; ++u) {
          onward(half + t + u, h[t + u], h[t + u + 1]);
          if (gate) {
            const ulonglong2 c2 = *reinterpret_cast<const ulonglong2*>(s_c + (half + t + u) * NP + 4 * p.sub);
#pragma unroll
            for (int c = 0; c < P::C; ++c) {
              float lo, hi;
              unf2(fma2(c2.x, h[t + u + 1][c][0], mul2(c2.y, h[t + u + 1][c][1])), lo, hi);
              acc[u * P::C + c] = lo + hi;
            }
          }
        }
        if (gate) {
          const int first = Sums::run(acc, p.sub);
          if (p.sub % Sums::SAME == 0) {
#pragma unroll
            for (int j = 0; j < Sums::LEFT; ++j) s_yp[(half + t + (first + j) / P::C) * P::YS + p.ch + (first + j) % P::C] = acc[j];
          }
        }
      }
      float acc[4];   // two sums for each of two (token, channel)
#pragma unroll
      for (int u = HALF - 1; u >= 0; --u) {
        const int t = half + u;
        const Pack<float2, P::C> q = load_pack<float2, P::C>(s_q + t * CH + p.ch);
        const Pack<float, P::C> dg = load_pack<float, P::C>(s_g + t * CH + p.ch);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(s_b + t * NP + 4 * p.sub);
        const ulonglong2 c2 = *reinterpret_cast<const ulonglong2*>(s_c + t * NP + 4 * p.sub);
        float v[8];
        uint64_t vb[2], vc[2];
#pragma unroll
        for (int c = 0; c < P::C; ++c) {
          const uint64_t step = f2(q.e[c].x, q.e[c].x), sx = f2(q.e[c].y, q.e[c].y), dout = f2(dg.e[c], dg.e[c]);
          const uint64_t g0 = fma2(dout, c2.x, r[c][0]), g1 = fma2(dout, c2.y, r[c][1]);
          const int at = u % UB * P::C + c;
          float lo, hi;
          unf2(fma2(g0, b.x, mul2(g1, b.y)), lo, hi);
          acc[at] = lo + hi;
          r[c][0] = mul2(ex2_pair(mul2(step, a2[c][0])), g0);
          r[c][1] = mul2(ex2_pair(mul2(step, a2[c][1])), g1);
          const uint64_t w0 = mul2(r[c][0], h[u][c][0]), w1 = mul2(r[c][1], h[u][c][1]);
          unf2(fma2(a2[c][0], w0, mul2(a2[c][1], w1)), lo, hi);
          acc[2 + at] = lo + hi;
          da[c][0] = fma2(step, w0, da[c][0]);
          da[c][1] = fma2(step, w1, da[c][1]);
          vb[0] = c == 0 ? mul2(sx, g0) : fma2(sx, g0, vb[0]);
          vb[1] = c == 0 ? mul2(sx, g1) : fma2(sx, g1, vb[1]);
          vc[0] = c == 0 ? mul2(dout, h[u + 1][c][0]) : fma2(dout, h[u + 1][c][0], vc[0]);
          vc[1] = c == 0 ? mul2(dout, h[u + 1][c][1]) : fma2(dout, h[u + 1][c][1], vc[1]);
        }
        if (u % UB == 0) {
          const int from = Sums::run(acc, p.sub);
          if (p.sub % Sums::SAME == 0) {
#pragma unroll
            for (int j = 0; j < Sums::LEFT; ++j)
              s_sum[(from + j) / 2 * S2 + (t + (from + j) % 2 / P::C) * P::YS + p.ch + (from + j) % P::C] = acc[j];
          }
        }
        unf2(vb[0], v[0], v[1]); unf2(vb[1], v[2], v[3]);
        unf2(vc[0], v[4], v[5]); unf2(vc[1], v[6], v[7]);
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
        if (u % TF == 0) {   // TF tokens are there: over the warps
          __syncthreads();
          for (int e = threadIdx.x; e < TF * 2 * NP; e += P::THREADS) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < P::WARPS; ++w) a += s_part[w * TF * 2 * NP + e];
            const int tt = t0 + t + e / (2 * NP);
            float* to = bc + (size_t)(tt - t_begin) * (2 * NP) + e % (2 * NP);
            if (tt < t_end) *to = first_turn ? a : *to + a;
          }
          __syncthreads();
        }
      }
    }
    float bias[V], skip[V];
    param(k.in.dt_bias, bias);
    param(k.in.skip, skip);
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      const int q = p.row + i * P::ROWS, t = t0 + q, at = q * CH + p.col;
      if (!p.col_on || t >= t_end) continue;
      float xv[V], dt[V], dout[V], s1[V], s2[V], o[V];
      ring.get(tile, 0, i, p, xv);
      ring.get(tile, 1, i, p, dt);
      unpack(load_pack<float, V>(s_g + at), dout);
      unpack(load_pack<float, V>(s_sum + q * P::YS + p.col), s1);
      unpack(load_pack<float, V>(s_sum + S2 + q * P::YS + p.col), s2);
      const Pack<float2, V> step = load_pack<float2, V>(s_q + at);
      const size_t out = ((size_t)p.b * s.S + t) * s.D + p.dcol;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        o[e] = fmaf(step.e[e].x, s1[e], skip[e] * dout[e]);
        dskip[e] = fmaf(dout[e], xv[e], dskip[e]);
      }
      store_pack<T, V>(static_cast<T*>(k.dx) + out, pack<T, V>(o));
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(xv[e], s1[e], s2[e] * kLn2);
      if (s.softplus) {
        float sg[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dt[e] += bias[e];
        logistic_v<T, V>(dt, sg);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] *= sg[e];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) dbias[e] += o[e];
      store_pack<T, V>(static_cast<T*>(k.ddt) + out, pack<T, V>(o));
      if (gate) {
        float zv[V], g[V], sg[V], yp[V];
        ring.get(tile, 2, i, p, zv);
        ring.get(tile, 3, i, p, g);
        unpack(load_pack<float, V>(s_yp + q * P::YS + p.col), yp);
        logistic_v<T, V>(zv, sg);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = g[e] * fmaf(skip[e], xv[e], yp[e]) * sg[e] * fmaf(zv[e], 1.f - sg[e], 1.f);
        store_pack<T, V>(static_cast<T*>(k.dz) + out, pack<T, V>(o));
      }
    }
    __syncthreads();   // the tile's arrays are free
  }
  const size_t row = (size_t)p.b * s.nseg + p.seg;
  ssm_put_states(k.part_a, p, row * s.D + p.d, da);
  if (k.dh0 != nullptr && p.seg == 0) ssm_store_states(k.dh0, s, p, (size_t)p.b * s.D + p.d, r);
  // dskip and ddt_bias: over the threads that share a channel
  float* s_x = reinterpret_cast<float*>(sm);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (p.row < SSM_TT) {
#pragma unroll
      for (int e = 0; e < V; ++e) s_x[p.row * CH + p.col + e] = which == 0 ? dskip[e] : dbias[e];
    }
    __syncthreads();
    constexpr int N_ROWS = P::ROWS < SSM_TT ? P::ROWS : SSM_TT;
    for (int c = threadIdx.x; c < CH; c += P::THREADS) {
      float a = 0.f;
#pragma unroll
      for (int q = 0; q < N_ROWS; ++q) a += s_x[q * CH + c];
      if (p.tile * CH + c < s.Dg) k.part_d[(row * 2 + which) * s.D + p.g * s.Dg + p.tile * CH + c] = a;
    }
    __syncthreads();
  }
}

template <typename T, int LN, int V>
__global__ void __launch_bounds__(SsmBwSmem<T, LN, V>::P::THREADS, SsmBwSmem<T, LN, V>::RESIDENT)
ssm_bw_kernel(SsmBw k, SsmDims s) {
  using P = typename SsmBwSmem<T, LN, V>::P;
  extern __shared__ __align__(16) char sm[];
  pdl_launch_dependents();
  pdl_wait();
#pragma unroll 1
  for (int turn = 0; turn < s.per_cta; ++turn) {
    const P p(s, s.nseg, 0, s.per_cta, turn);
    if (p.tile < s.tiles) ssm_bw_tile<T, LN, V>(k, s, p, turn == 0, sm);
  }
}

// The sums over CTAs, in their order: db and dc over the channel tiles, da, dskip and ddt_bias over sequences and segments.
struct SsmSums {
  const float *part_bc, *part_a, *part_d;
  void *db, *dc;                       // (B, S, G, N)
  float *da, *dskip, *ddt_bias;        // dskip, ddt_bias may be null
  int NP;
  size_t n_bc, n_a, n_d;               // threads of each kind: 2 G rows seg NP of this launch's rows, D NP, 2 D
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
    const size_t per_part = (size_t)s.rows * s.seg, at = k % per_part;
    const int g = (int)(k / per_part), row = s.row0 + (int)(at / s.seg), t = row % s.nseg * s.seg + (int)(at % s.seg);
    if (n >= s.N || row >= s.B * s.nseg || t >= s.S) return;
    const size_t tok = (size_t)(row / s.nseg) * s.S + t;
    const float* src = q.part_bc + ((size_t)g * s.parts * per_part + at) * 2 * q.NP + which * q.NP + n;
    float a = 0.f;
    for (int i = 0; i < s.parts; ++i) a += src[i * per_part * 2 * q.NP];
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
  if (id >= q.n_d) return;
  const int which = id >= (size_t)s.D;
  const size_t d = id - (which ? s.D : 0);
  float* out = which ? q.ddt_bias : q.dskip;
  if (out == nullptr) return;
  float a = 0.f;
  for (int t = 0; t < rows; ++t) a += q.part_d[((size_t)t * 2 + which) * s.D + d];
  out[d] = a;
}

// ---- launchers ----------------------------------------------------------------------------------------
SsmDims ssm_dims(int B, int S, int D, int N, int G, bool softplus, const long long* strides, bool backward, int dtype);
bool ssm_tokens_ok(const long long* strides);
template <typename T> bool ssm_vec(const SsmIn& in, const SsmDims& s, const void* dy, const void* y);
template <typename T> bool ssm_pairs(const SsmIn& in, const SsmDims& s);

struct SsmBwLayout { size_t bc, a, d, g, sum, end; };
static SsmBwLayout ssm_bw_layout(const SsmDims& s) {
  const size_t np = ssm_padded(s.N), rows = (size_t)s.B * s.nseg;
  SsmBwLayout l{};
  l.bc = 0;
  l.a = align_up(l.bc + (size_t)s.G * s.parts * s.rows * s.seg * 2 * np * sizeof(float), 256);
  l.d = align_up(l.a + rows * s.D * np * sizeof(float), 256);
  l.g = align_up(l.d + rows * 2 * s.D * sizeof(float), 256);
  l.sum = align_up(l.g + (s.nseg > 1 ? rows * s.D * np * sizeof(float) : 0), 256);
  l.end = align_up(l.sum + (s.nseg > 1 ? rows * s.D * sizeof(float) : 0), 256);
  return l;
}
// (for every element type)
size_t ssm_bw_bytes(int B, int S, int D, int N, int G) {
  size_t most = 0;
  for (const int dtype : {MLSTM_F32, MLSTM_BF16}) most = std::max(most, ssm_bw_layout(ssm_dims(B, S, D, N, G, false, nullptr, true, dtype)).end);
  return most;
}
ScanSlots ssm_bw_slots(int lanes, int dtype) {
  MLSTM_DTYPE_SWITCH(dtype, T, SSM_LANES_SWITCH(lanes, LN, return (ScanSlots{SsmBwSmem<T, LN, 4>::RESIDENT, SsmBwLocalSmem<T, LN, 4>::RESIDENT});))
  return ScanSlots{1, 1};
}

template <typename T, int LN, int V>
static int ssm_bw_t(const SsmBw& k, SsmDims s, SsmSums q, cudaStream_t st) {
  if (s.nseg > 1) {   // the first segment leaves nothing to another
    const unsigned local = (unsigned)s.B * s.G * s.tiles * (s.nseg - 1);
    if (int rc = ssm_launch(ssm_bw_local_kernel<T, LN, V>, 256 / SSM_BW_LOCAL_C, SsmBwLocalSmem<T, LN, V>::BYTES, local <= pdl_max_ctas(), local, st, k, s, s.nseg - 1)) return rc;
  }
  const int all = s.B * s.nseg;
  for (; s.row0 < all; s.row0 += s.rows) {
    const int rows = all - s.row0 < s.rows ? all - s.row0 : s.rows;
    const unsigned grid = (unsigned)s.G * s.parts * rows;
    if (int rc = ssm_launch(ssm_bw_kernel<T, LN, V>, 256 / SSM_BW_C, SsmBwSmem<T, LN, V>::BYTES, grid <= pdl_max_ctas(), grid, st, k, s)) return rc;
    SsmSums sums = q;
    if (s.row0 + s.rows < all) sums.n_a = sums.n_d = 0;   // these when all of their parts are there
    const size_t threads = sums.n_bc + sums.n_a + sums.n_d, ctas = (threads + 255) / 256;
    if (int rc = launch_pdl(ctas <= pdl_max_ctas(), ssm_bw_sums_kernel<T>, (unsigned)ctas, 256, 0, st, sums, s)) return rc;
  }
  return MLSTM_OK;
}

int launch_ssm_bw(const SsmIn& in, const long long* strides, const void* dy, const long long* gs, const float* dh_last, const float* ckpt, void* dx,
                  void* ddt, void* dz, void* db, void* dc, float* da, float* dskip, float* ddt_bias, float* dh0, void* workspace, int B, int S, int D,
                  int N, int G, bool softplus, int dtype, cudaStream_t st) {
  if (!ssm_sizes_ok(B, S, D, N, G) || !ssm_tokens_ok(strides) || gs[1] < 0 || gs[1] >= (1ll << 29)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_SCAN, st);
  SsmDims s = ssm_dims(B, S, D, N, G, softplus, strides, true, dtype);
  s.gb = gs[0]; s.gt = (int)gs[1];
  const int lanes = ssm_lanes(N), np = ssm_padded(N);
  const SsmBwLayout l = ssm_bw_layout(s);
  char* w = static_cast<char*>(workspace);
  auto at = [&](size_t o) { return reinterpret_cast<float*>(w + o); };
  const SsmBw k{in, dy, dh_last, ckpt, dx, ddt, dz, dh0, at(l.bc), at(l.a), at(l.d), at(l.g), at(l.sum)};
  const SsmSums q{k.part_bc, k.part_a, k.part_d, db, dc, da, dskip, ddt_bias, np, (size_t)2 * G * s.rows * s.seg * np, (size_t)D * np, 2 * (size_t)D};
  if ((q.n_bc + q.n_a + q.n_d + 255) / 256 >= (1ull << 31)) return MLSTM_ERR_SHAPE;
  MLSTM_DTYPE_SWITCH(dtype, T,
    s.pairs = ssm_pairs<T>(in, s);
    const bool vec = ssm_vec<T>(in, s, dy, dx) && ssm_vec<T>(in, s, ddt, dz);
    SSM_LANES_SWITCH(lanes, LN, return vec ? ssm_bw_t<T, LN, 4>(k, s, q, st) : ssm_bw_t<T, LN, 1>(k, s, q, st);))
  return MLSTM_ERR_DTYPE;
}

}  // namespace mlstm
