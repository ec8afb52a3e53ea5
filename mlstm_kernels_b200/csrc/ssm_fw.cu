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
// 16384 x 2048 channels of 16 states in bf16, 23 segments: 385 us; alone, with cold caches, the end states take 174 (special functions
// 81 % busy) and the scan 231 (70 %).  1024 channels, whole in one segment: 2083, in 64 segments 210.
#include <algorithm>

#include "ssm.cuh"

namespace mlstm {

// Two channels to a thread: b and c come from shared memory once for both, at 128 bytes a clock and SM.
constexpr int SSM_FW_C = 2;

struct SsmFw {
  SsmIn in;
  void* y;
  float* h_last;       // (B, D, N) or null
  float* ckpt;         // (B, nt, D, NP): the state before every tile, or null
  float* loc_h;        // (B, nseg, D, NP) end states of the segments, from an empty start
  float* loc_sum;      // (B, nseg, D) sums of their steps
};

// Shared memory of the forward, in bytes
template <typename T, int LN, int V, bool LOCAL> struct SsmFwSmem {
  using P = SsmPlace<LN, V, SSM_FW_C>;
  using Ring = SsmRing<T, P, V, LOCAL ? 2 : 3, LOCAL ? 1 : 2>;
  static constexpr size_t Q = 0, B = Q + sizeof(float2) * SSM_TT * P::CH, C = B + sizeof(float) * SSM_TT * P::NP,
                          Y = C + (LOCAL ? 0 : sizeof(float) * SSM_TT * P::NP), X = Y + (LOCAL ? 0 : sizeof(float) * SSM_TT * P::YS),
                          BYTES = X + Ring::BYTES;
  static constexpr int RESIDENT = scan_resident(BYTES, 5);
};

// LOCAL: only a segment's own end state and sum of steps
template <typename T, int LN, int V, bool LOCAL>
__global__ void __launch_bounds__(SsmFwSmem<T, LN, V, LOCAL>::P::THREADS, SsmFwSmem<T, LN, V, LOCAL>::RESIDENT)
ssm_fw_kernel(SsmFw k, SsmDims s, int nseg) {
  using Mem = SsmFwSmem<T, LN, V, LOCAL>;
  using P = typename Mem::P;
  using Ring = typename Mem::Ring;
  using Sums = LaneSums<LN>;
  constexpr int CH = P::CH, AHEAD = Ring::STAGES - 1;
  extern __shared__ __align__(16) char sm[];
  float2* s_d = reinterpret_cast<float2*>(sm + Mem::Q);          // (step, step x)
  float *s_b = reinterpret_cast<float*>(sm + Mem::B), *s_c = reinterpret_cast<float*>(sm + Mem::C), *s_y = reinterpret_cast<float*>(sm + Mem::Y);
  const Ring ring{reinterpret_cast<T*>(sm + Mem::X)};            // x, dt, z; b, c
  pdl_launch_dependents();
  pdl_wait();
  const P p(s, nseg, 0);
  uint64_t a2[P::C][P::H], h[P::C][P::H];
  float sum[P::C];
#pragma unroll
  for (int c = 0; c < P::C; ++c) sum[c] = 0.f;
  ssm_rates(k.in.a, s, p, a2);
  ssm_load_states(LOCAL ? nullptr : k.in.h0, s, p, (size_t)p.b * s.D + p.d, h);
  if (!LOCAL) ssm_fold<false>(k.loc_h, k.loc_sum, 0, p.seg, s, p, a2, h);
  float bias[V], skip[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = k.in.dt_bias != nullptr && p.col_on ? k.in.dt_bias[p.dcol + i] : 0.f;
    skip[i] = !LOCAL && k.in.skip != nullptr && p.col_on ? k.in.skip[p.dcol + i] : 0.f;
  }
  const int t_begin = p.seg * s.seg, t_end = min(s.S, t_begin + s.seg);
  const bool gate = !LOCAL && k.in.z != nullptr;
  const SsmSource from_x = ssm_source<T>(k.in.x, p.b * s.xb + p.dcol, s.xt), from_dt = ssm_source<T>(k.in.dt, p.b * s.db + p.dcol, s.dt),
                  from_z = ssm_source<T>(k.in.z, p.b * s.zb + p.dcol, s.zt), from_b = Ring::source_bc(k.in.b, p, s.bb, s.bt, s.bg),
                  from_c = Ring::source_bc(k.in.c, p, s.cb, s.ct, s.cg);
  auto fetch = [&](int t0) {
    if (t0 < t_end) {
      ring.copy(s, p, t0, 0, from_x);
      ring.copy(s, p, t0, 1, from_dt);
      if (gate) ring.copy(s, p, t0, 2, from_z);
      ring.copy_bc(s, p, t0, 0, from_b);
      if (!LOCAL) ring.copy_bc(s, p, t0, 1, from_c);
    }
    cp_commit();
  };
  ring.clear(s, p);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(t_begin + i * SSM_TT);
  for (int t0 = t_begin; t0 < t_end; t0 += SSM_TT) {
    const int tile = t0 / SSM_TT;
    cp_wait<AHEAD - 1>();
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      const int r = p.row + i * P::ROWS;
      if (r >= SSM_TT) continue;
      float dt[V], step[V], xv[V];
      ring.get(tile, 0, i, p, xv);
      ring.get(tile, 1, i, p, dt);
      ssm_step_v<T, V>(dt, bias, s.softplus, t0 + r >= t_end, step);
      Pack<float2, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.e[e] = make_float2(step[e], step[e] * xv[e]);
      store_pack<float2, V>(s_d + r * CH + p.col, o);
    }
    ring.put(tile, 0, s_b);
    if (!LOCAL) ring.put(tile, 1, s_c);
    __syncthreads();
    fetch(t0 + AHEAD * SSM_TT);
    if (!LOCAL && k.ckpt != nullptr) ssm_put_states(k.ckpt, p, ((size_t)p.b * s.nt + t0 / SSM_TT) * s.D + p.d, h);
    constexpr int U = 4 / P::C;   // tokens whose sums over the states are taken together
#pragma unroll(LOCAL ? 2 : 16)
    for (int t = 0; t < SSM_TT; t += U) {
      float acc[4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Pack<float2, P::C> q = load_pack<float2, P::C>(s_d + (t + u) * CH + p.ch);
        const Pack<uint64_t, P::H> b = ssm_token(s_b, t + u, p);
#pragma unroll
        for (int c = 0; c < P::C; ++c) {
          const uint64_t step = f2(q.e[c].x, q.e[c].x), sx = f2(q.e[c].y, q.e[c].y);
#pragma unroll
          for (int i = 0; i < P::H; ++i) h[c][i] = fma2(ex2_pair(mul2(step, a2[c][i])), h[c][i], mul2(sx, b.e[i]));
          if (LOCAL) sum[c] += q.e[c].x;
        }
        if (!LOCAL) {
          const Pack<uint64_t, P::H> c2 = ssm_token(s_c, t + u, p);
#pragma unroll
          for (int c = 0; c < P::C; ++c) {
            uint64_t v = mul2(c2.e[0], h[c][0]);
#pragma unroll
            for (int i = 1; i < P::H; ++i) v = fma2(c2.e[i], h[c][i], v);
            float lo, hi;
            unf2(v, lo, hi);
            acc[u * P::C + c] = lo + hi;
          }
        }
      }
      if (!LOCAL) {
        const int first = Sums::run(acc, p.sub);
        if (p.sub % Sums::SAME == 0) {
#pragma unroll
          for (int j = 0; j < Sums::LEFT; ++j) s_y[(t + (first + j) / P::C) * P::YS + p.ch + (first + j) % P::C] = acc[j];
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
      T* yp = static_cast<T*>(k.y) + (size_t)p.b * s.S * s.D + p.dcol;
#pragma unroll
      for (int i = 0; i < P::ITEMS; ++i) {
        const int r = p.row + i * P::ROWS, t = t0 + r;
        if (!p.col_on || t >= t_end) continue;
        float xv[V], o[V];
        ring.get(tile, 0, i, p, xv);
        const Pack<float, V> sums = load_pack<float, V>(s_y + r * P::YS + p.col);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(skip[e], xv[e], sums.e[e]);
        if (gate) {
          float zv[V], sg[V];
          ring.get(tile, 2, i, p, zv);
          logistic_v<T, V>(zv, sg);
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] *= zv[e] * sg[e];
        }
        store_pack<T, V>(yp + (size_t)t * s.D, pack<T, V>(o));
      }
    }
  }
  if (LOCAL) {
    const size_t at = ((size_t)p.b * s.nseg + p.seg) * s.D + p.d;
    ssm_put_states(k.loc_h, p, at, h);
#pragma unroll
    for (int c = 0; c < P::C; ++c)
      if (p.on[c] && p.sub == 0) k.loc_sum[at + c] = sum[c];
  } else if (k.h_last != nullptr && p.seg == s.nseg - 1) {
    ssm_store_states(k.h_last, s, p, (size_t)p.b * s.D + p.d, h);
  }
}

// One token: bound by the states, in and out once each, 16 bytes at a time (VEC; else element by element).  LN lanes share a channel,
// each with J times four of its states, LN apart from one another, so that a warp's accesses are whole sectors; what is done once
// for a channel (some 150 instructions) is done by few lanes.
constexpr int SSM_STEP_THREADS = 128;
template <typename T, int LN, int J, bool VEC>
__global__ void __launch_bounds__(SSM_STEP_THREADS)
ssm_step_kernel(const T* x, const T* dt, const T* z, const T* b, const T* c, const float* a, const float* skip, const float* dt_bias,
                const float* h, T* y, float* h_new, int tiles, int D, int N, int G, bool softplus) {
  constexpr int CH = SSM_STEP_THREADS / LN;
  pdl_launch_dependents();
  pdl_wait();
  const int sub = threadIdx.x % LN;
  const unsigned bi = blockIdx.x / (unsigned)tiles;
  const int d = (int)(blockIdx.x - bi * (unsigned)tiles) * CH + threadIdx.x / LN;
  const bool on = d < D;
  const int dc = on ? d : 0, g = G == 1 ? 0 : (int)((unsigned)dc / ((unsigned)D / (unsigned)G));
  const size_t row = (size_t)bi * D + dc, bc = ((size_t)bi * G + g) * N;
  const float *hr = h + row * N, *ar = a + (size_t)dc * N;
  float hv[J][4], av[J][4], bv[J][4], cv[J][4];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int n = 4 * (sub + j * LN);
#pragma unroll
    for (int i = 0; i < 4; ++i) hv[j][i] = av[j][i] = bv[j][i] = cv[j][i] = 0.f;
    if (VEC) {
      if (n < N) {
        const float4 q = ld_stream(reinterpret_cast<const float4*>(hr + n));
        hv[j][0] = q.x; hv[j][1] = q.y; hv[j][2] = q.z; hv[j][3] = q.w;
        unpack(load_pack<float, 4>(ar + n), av[j]);
        unpack(load_pack<T, 4>(b + bc + n), bv[j]);
        unpack(load_pack<T, 4>(c + bc + n), cv[j]);
      }
    } else {
      ssm_load<4>(hr, N, n, hv[j]);
      ssm_load<4>(ar, N, n, av[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n + i >= N) continue;
        bv[j][i] = to_f32(b[bc + n + i]);
        cv[j][i] = to_f32(c[bc + n + i]);
      }
    }
  }
  const float raw[1] = {to_f32(dt[row])}, bias[1] = {dt_bias != nullptr ? dt_bias[dc] : 0.f};
  const float xv = to_f32(x[row]), zv = z != nullptr ? to_f32(z[row]) : 0.f, sk = skip != nullptr ? skip[dc] : 0.f;
  float st[1], acc = 0.f;
  ssm_step_v<T, 1>(raw, bias, softplus, false, st);
  const float sx = st[0] * xv, s2 = st[0] * kLog2e;
  float* out = h_new + row * N;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int n = 4 * (sub + j * LN);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hv[j][i] = fmaf(ex2(s2 * av[j][i]), hv[j][i], sx * bv[j][i]);
      acc = fmaf(cv[j][i], hv[j][i], acc);
    }
    if (VEC) {
      if (on && n < N) __stcs(reinterpret_cast<float4*>(out + n), make_float4(hv[j][0], hv[j][1], hv[j][2], hv[j][3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (on && n + i < N) out[n + i] = hv[j][i];
    }
  }
#pragma unroll
  for (int o = LN / 2; o >= 1; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (on && sub == 0) {
    const float v = fmaf(sk, xv, acc);
    y[row] = from_f32<T>(z != nullptr ? v * (zv * logistic_f<T>(zv)) : v);
  }
}

// ---- launchers ----------------------------------------------------------------------------------------
bool ssm_sizes_ok(int B, int S, int D, int N, int G) {
  if (B <= 0 || S <= 0 || D <= 0 || N <= 0 || N > SSM_MAX_N || G <= 0 || D % G != 0) return false;
  if (S > (1 << 30) || (long long)D * N >= (1ll << 31)) return false;
  const int ch = ssm_tile_channels(N), Dg = D / G;
  return (long long)B * G * ceil_div(Dg, ch) * 64 < (1ll << 31);
}

// Token strides are 32-bit numbers of bytes in the kernels.
bool ssm_tokens_ok(const long long* st) {
  const long long q[] = {st[1], st[3], st[5], st[7], st[10]};
  for (const long long t : q)
    if (t < 0 || t >= (1ll << 29)) return false;
  return true;
}

size_t ssm_ckpt_bytes(int B, int S, int D, int N) { return (size_t)B * ceil_div(S, SSM_TT) * D * ssm_padded(N) * sizeof(float); }

static ScanSlots ssm_fw_slots(int lanes, int dtype) {
  MLSTM_DTYPE_SWITCH(dtype, T, SSM_LANES_SWITCH(lanes, LN, return (ScanSlots{SsmFwSmem<T, LN, 4, false>::RESIDENT, SsmFwSmem<T, LN, 4, true>::RESIDENT});))
  return ScanSlots{1, 1};
}
constexpr int SSM_MAX_PARTS = 64;
constexpr size_t SSM_PART_BYTES = 64 << 20;
SsmDims ssm_dims(int B, int S, int D, int N, int G, bool softplus, const long long* st, bool backward, int dtype) {
  SsmDims s{};
  s.B = B; s.S = S; s.D = D; s.N = N; s.G = G;
  s.Dg = D / G;
  s.tiles = ceil_div(s.Dg, ssm_tile_channels(N));
  s.nt = ceil_div(S, SSM_TT);
  // Each CTA of the backward writes its channels' sums of db and dc, 2 NP values a token: no more than 64 CTAs to a group (8192
  // channels of 16 states: 128 tiles in 64 CTAs).
  s.per_cta = backward ? ceil_div(s.tiles, SSM_MAX_PARTS) : 1;
  s.parts = ceil_div(s.tiles, s.per_cta);
  const ScanSlots held = backward ? ssm_bw_slots(ssm_lanes(N), dtype) : ssm_fw_slots(ssm_lanes(N), dtype);
  const int n = scan_segments((long long)B * G * s.parts, s.per_cta, (long long)B * G * s.tiles, s.nt, ssm_padded(N), backward, held, sm_count());
  s.seg = ceil_div(s.nt, n) * SSM_TT;
  if (backward) {
    // With many states or groups these sums are more than all other memory of the call together (128 states in 8 groups of 512
    // channels: 512 KB a token).  They are given 64 MB (half of L2), or twice what the states take that the forward kept, and the
    // segments go in as many launches as that takes, each followed by the sums over its CTAs; a segment is short enough to fit.
    const size_t kept = 2 * ssm_ckpt_bytes(B, S, D, N), room = kept > SSM_PART_BYTES ? kept : SSM_PART_BYTES;
    const size_t token = (size_t)G * s.parts * 2 * ssm_padded(N) * sizeof(float);
    while (s.seg > SSM_TT && s.seg * token > room) s.seg = ceil_div(s.seg / SSM_TT, 2) * SSM_TT;
    s.nseg = ceil_div(S, s.seg);
    const long long rows = (long long)B * s.nseg, fit = (long long)(room / (s.seg * token)), most = (size_t)B * S * token <= room ? rows : fit < 1 ? 1 : std::min(rows, fit);
    s.rows = (int)most;
    if (most < rows) {   // of the numbers just below, the one whose launches leave least of the GPU empty at their ends
      const long long ctas = (long long)G * s.parts, slots = (long long)held.whole * sm_count();
      auto rounds = [&](long long r) { return (rows + r - 1) / r * ((r * ctas + slots - 1) / slots); };
      for (long long r = most - 1; r > 0 && 2 * r >= most && r > most - 64; --r)
        if (rounds(r) < rounds(s.rows)) s.rows = (int)r;
    }
  }
  s.nseg = ceil_div(S, s.seg);
  s.softplus = softplus;
  s.pairs = false;
  if (st != nullptr) {
    s.xb = st[0]; s.xt = (int)st[1]; s.db = st[2]; s.dt = (int)st[3]; s.zb = st[4]; s.zt = (int)st[5];
    s.bb = st[6]; s.bt = (int)st[7]; s.bg = st[8]; s.cb = st[9]; s.ct = (int)st[10]; s.cg = st[11];
  }
  return s;
}

// (for every element type)
size_t ssm_fw_bytes(int B, int S, int D, int N, int G) {
  int nseg = 1;
  for (const int dtype : {MLSTM_F32, MLSTM_BF16}) nseg = std::max(nseg, ssm_dims(B, S, D, N, G, false, nullptr, false, dtype).nseg);
  const size_t rows = nseg > 1 ? (size_t)B * nseg * D : 0;
  return rows * ssm_padded(N) * sizeof(float) + rows * sizeof(float);
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
// b and c two elements at a time
template <typename T> bool ssm_pairs(const SsmIn& in, const SsmDims& s) {
  if (s.N % 2 != 0 || !fits_access(in.b, 2 * sizeof(T)) || !fits_access(in.c, 2 * sizeof(T))) return false;
  const long long strides[] = {s.bb, s.bt, s.bg, s.cb, s.ct, s.cg};
  for (const long long q : strides)
    if (q % 2 != 0) return false;
  return true;
}
template bool ssm_pairs<float>(const SsmIn&, const SsmDims&);
template bool ssm_pairs<__nv_bfloat16>(const SsmIn&, const SsmDims&);
template bool ssm_pairs<__half>(const SsmIn&, const SsmDims&);
template bool ssm_vec<float>(const SsmIn&, const SsmDims&, const void*, const void*);
template bool ssm_vec<__nv_bfloat16>(const SsmIn&, const SsmDims&, const void*, const void*);
template bool ssm_vec<__half>(const SsmIn&, const SsmDims&, const void*, const void*);

template <typename T, int LN, int V>
static int ssm_fw_t(const SsmFw& k, const SsmDims& s, cudaStream_t st) {
  const unsigned per_seg = (unsigned)s.B * s.G * s.tiles, grid = per_seg * s.nseg;
  const bool overlap = grid <= pdl_max_ctas();
  if (s.nseg > 1)   // the last segment leaves nothing to another
    if (int rc = ssm_launch(ssm_fw_kernel<T, LN, V, true>, 256 / SSM_FW_C, SsmFwSmem<T, LN, V, true>::BYTES, overlap, per_seg * (s.nseg - 1), st, k, s, s.nseg - 1)) return rc;
  return ssm_launch(ssm_fw_kernel<T, LN, V, false>, 256 / SSM_FW_C, SsmFwSmem<T, LN, V, false>::BYTES, overlap, grid, st, k, s, s.nseg);
}

int launch_ssm_fw(const SsmIn& in, const long long* strides, void* y, float* h_last, float* ckpt, void* workspace, int B, int S, int D, int N, int G,
                  bool softplus, int dtype, cudaStream_t st) {
  if (!ssm_sizes_ok(B, S, D, N, G) || !ssm_tokens_ok(strides)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_SCAN, st);
  SsmDims s = ssm_dims(B, S, D, N, G, softplus, strides, false, dtype);
  SsmFw k{in, y, h_last, ckpt, nullptr, nullptr};
  if (s.nseg > 1) {
    k.loc_h = static_cast<float*>(workspace);
    k.loc_sum = k.loc_h + (size_t)B * s.nseg * D * ssm_padded(N);
  }
  MLSTM_DTYPE_SWITCH(dtype, T,
    const bool vec = ssm_vec<T>(in, s, nullptr, y);
    s.pairs = ssm_pairs<T>(in, s);
    SSM_LANES_SWITCH(ssm_lanes(N), LN, return vec ? ssm_fw_t<T, LN, 4>(k, s, st) : ssm_fw_t<T, LN, 1>(k, s, st);))
  return MLSTM_ERR_DTYPE;
}

int launch_ssm_step(const void* x, const void* dt, const void* z, const void* b, const void* c, const float* a, const float* skip, const float* dt_bias,
                    const float* h, void* y, float* h_new, int B, int D, int N, int G, bool softplus, int dtype, cudaStream_t st) {
  if (!ssm_sizes_ok(B, 1, D, N, G)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_STEP, st);
  const int lanes = N <= 4 ? 1 : N <= 16 ? 2 : N <= 64 ? 4 : 8, tiles = ceil_div(D, SSM_STEP_THREADS / lanes);
  const size_t grid = (size_t)B * tiles;
  if (grid >= (1ull << 31)) return MLSTM_ERR_SHAPE;
  const size_t four = 4 * dtype_size(dtype);
  const bool vec = N % 4 == 0 && fits_access(a, 16) && fits_access(h, 16) && fits_access(h_new, 16) && fits_access(b, four) && fits_access(c, four);
#define RUN(LN, J)                                                                                                                                \
  return launch_pdl(grid <= 2 * pdl_max_ctas(), vec ? ssm_step_kernel<T, LN, J, true> : ssm_step_kernel<T, LN, J, false>, (unsigned)grid,         \
                    SSM_STEP_THREADS, 0, st, (const T*)x, (const T*)dt, (const T*)z, (const T*)b, (const T*)c, a, skip, dt_bias, h, (T*)y, h_new, \
                    tiles, D, N, G, softplus)
  MLSTM_DTYPE_SWITCH(dtype, T, if (N <= 4) RUN(1, 1); if (N <= 8) RUN(2, 1); if (N <= 16) RUN(2, 2); if (N <= 32) RUN(4, 2); if (N <= 64) RUN(4, 4); RUN(8, 4);)
#undef RUN
  return MLSTM_ERR_DTYPE;
}

}  // namespace mlstm
