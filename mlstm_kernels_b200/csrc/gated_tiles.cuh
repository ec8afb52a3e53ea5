// Gated linear recurrence over sequences: forward and backward kernels of one element type (formulas: gated.cuh).
//
// A run of tokens acts on the state before it as h -> A h + H (A the product of its factors, H its own end state), and two runs after
// one another as A2 A1, A2 H1 + H2.  A thread takes GATED_CK tokens of a few channels in registers, the warps of a CTA take runs that
// follow one another: a unit (gated_units.h).  One pass over the data: every thread reduces its run to (A, H), these are exchanged in
// shared memory, the unit's first warp finds the state in front of the unit, every thread that in front of its run, and takes its tokens
// again out of its registers.
//
// Between units the states go through global memory.  CTAs take units in the order of their numbers, by a counter; what a unit waits
// for has a lower number, so that a CTA that runs has it or has done it: no unit waits for one that is not under way.  A unit
// publishes its own (A, H) as soon as it has it; the state in front of a group of units is published by the last unit of the group
// before.  A unit waits for the state in front of its group and joins the runs from there to itself, always in that order: results
// do not depend on who ran when.  Waits are bounded (gated_wait).
//
// The backward is the same in the other direction, on a_t (dyh_t + .): the forward has kept the state in front of every run, so that
// the states are recomputed without an exchange.
#pragma once
#include <algorithm>

#include "gated.cuh"

namespace mlstm {

// What is there, known when a kernel is compiled, or when it is called (for channels that come one by one)
template <bool RATE, int SCALE, bool I, bool Z> struct GatedFixed {
  __host__ __device__ static constexpr bool rate() { return RATE; }
  __host__ __device__ static constexpr int scale() { return SCALE; }
  __host__ __device__ static constexpr bool i() { return I; }
  __host__ __device__ static constexpr bool z() { return Z; }
};
struct GatedAny {
  bool rate_, i_, z_;
  int scale_;
  __device__ bool rate() const { return rate_; }
  __device__ int scale() const { return scale_; }
  __device__ bool i() const { return i_; }
  __device__ bool z() const { return z_; }
};

constexpr int GL = GATED_CK;

// ---- joining runs -------------------------------------------------------------------------------------
struct Run { uint64_t A, H; };   // of two channels
__device__ __forceinline__ Run no_tokens() { return Run{dup2(1.f), 0}; }
__device__ __forceinline__ Run then(Run first, Run second) { return Run{mul2(second.A, first.A), fma2(second.A, first.H, second.H)}; }
__device__ __forceinline__ uint64_t through(Run r, uint64_t h) { return fma2(r.A, h, r.H); }

// ---- units --------------------------------------------------------------------------------------------
// Code of the first wait that ran out since it was last asked for (0: none), read by the host
static __device__ int g_gated_status = 0;
constexpr unsigned kGatedWaitLimit = 1u << 24;   // polls: some seconds

__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// The lanes of a warp wait for a flag each (null: for none).  After kGatedWaitLimit polls, or once another wait of this launch has
// run out, they go on without: the results are wrong, the status says so, and every CTA ends.
__device__ __forceinline__ void gated_wait(const unsigned* flag, unsigned* gave_up) {
  bool there = flag == nullptr;
#pragma unroll 1
  for (unsigned n = 0; n < kGatedWaitLimit; ++n) {
    there = there || load_acquire(flag) != 0;
    if (__all_sync(0xffffffffu, there)) return;
    if ((n & 255) == 255 && __any_sync(0xffffffffu, load_acquire(gave_up) != 0)) return;
    __nanosleep(20);
  }
  if ((threadIdx.x & 31) == 0) {
    atomicExch(gave_up, 1u);
    atomicCAS(&g_gated_status, 0, 301);
  }
}
__device__ __forceinline__ void gated_publish(unsigned* flag) {   // what the warp has written
  __threadfence();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flag), "r"(1u) : "memory");
}

struct Unit { int k, chain, b, block; };   // its place in the chain (BACK: from the end), and the chain's
__device__ __forceinline__ Unit unit_of(int u, const GatedDims& q) {
  Unit o;
  o.k = q.chains(u);
  o.chain = u - o.k * (int)q.chains.d;
  o.b = q.blocks(o.chain);
  o.block = o.chain - o.b * (int)q.blocks.d;
  return o;
}

template <int P> struct alignas(16) GatedShared {
  Run part[GATED_WARPS][P][32];          // the warps' runs
  uint64_t start[P][32];                 // the state in front of the unit
  uint64_t drate[GATED_WARPS][32];       // (backward) sums of the unit before
  int unit[2];
};
// The next unit: by the counter, or, where no unit waits for another, every gridDim-th
__device__ __forceinline__ int take_unit(const GatedDims& q, int turn) {
  return q.ticket != nullptr ? (int)min(atomicAdd(q.ticket, 1u), 0x7fffffffu) : min((long long)blockIdx.x + (long long)turn * gridDim.x, 0x7fffffffll);
}

// The first warp, behind the barrier behind which all parts are there: finds the state in front of the unit, for all warps, and gives
// the units after it what they need.  first: the state in front of the chain; returns the state behind the unit.
template <bool BACK, int P> __device__ __forceinline__ void gated_unit_start(GatedShared<P>& sh, const GatedDims& q, const Unit& u, const uint64_t (&first)[P],
                                                                               uint64_t (&end)[P]) {
  const int lane = threadIdx.x & 31, W = blockDim.x >> 5;
  Run all[P];
#pragma unroll
  for (int k = 0; k < P; ++k) all[k] = sh.part[BACK ? W - 1 : 0][k][lane];
  for (int n = 1; n < W; ++n)
#pragma unroll
    for (int k = 0; k < P; ++k) all[k] = then(all[k], sh.part[BACK ? W - 1 - n : n][k][lane]);
  uint64_t h[P];
#pragma unroll
  for (int k = 0; k < P; ++k) h[k] = first[k];
  if (q.nt > 1) {
    const int group = u.k / q.group, pos = u.k - group * q.group;
    const long long in_chain = (long long)u.chain * q.nt + u.k - pos;   // the group's first unit
    Run* const agg = static_cast<Run*>(q.agg) + in_chain * (P * 32) + lane;
    uint64_t* const state = static_cast<uint64_t*>(q.state) + ((long long)u.chain * q.groups + group) * (P * 32) + lane;
    unsigned* const state_flag = q.state_flag + (long long)u.chain * q.groups + group;
    const bool last = pos == q.group - 1, more = u.k < q.nt - 1;
    if (more && !last) {
#pragma unroll
      for (int k = 0; k < P; ++k) __stcg(reinterpret_cast<ulonglong2*>(agg + (pos * P + k) * 32), make_ulonglong2(all[k].A, all[k].H));
      gated_publish(q.agg_flag + in_chain + pos);
    }
    gated_wait(lane < pos ? q.agg_flag + in_chain + lane : lane == 31 && group > 0 ? state_flag : nullptr, q.gave_up);
    if (group > 0) {
#pragma unroll
      for (int k = 0; k < P; ++k) h[k] = __ldcg(reinterpret_cast<const unsigned long long*>(state + k * 32));
    }
#pragma unroll 4
    for (int n = 0; n < pos; ++n)
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const ulonglong2 r = __ldcg(reinterpret_cast<const ulonglong2*>(agg + (n * P + k) * 32));
        h[k] = through(Run{r.x, r.y}, h[k]);
      }
#pragma unroll
    for (int k = 0; k < P; ++k) end[k] = through(all[k], h[k]);
    if (more && last) {
#pragma unroll
      for (int k = 0; k < P; ++k) __stcg(reinterpret_cast<unsigned long long*>(state + (P + k) * 32), (unsigned long long)end[k]);
      gated_publish(state_flag + 1);
    }
  } else {
#pragma unroll
    for (int k = 0; k < P; ++k) end[k] = through(all[k], h[k]);
  }
#pragma unroll
  for (int k = 0; k < P; ++k) sh.start[k][lane] = h[k];
}
// What the warps in front of this one make of the state in front of the unit
template <bool BACK, int P> __device__ __forceinline__ void gated_front(const GatedShared<P>& sh, Run (&front)[P]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < P; ++k) front[k] = no_tokens();
  for (int n = 0; n < (BACK ? W - 1 - warp : warp); ++n)
#pragma unroll
    for (int k = 0; k < P; ++k) front[k] = then(front[k], sh.part[BACK ? W - 1 - n : n][k][lane]);
}

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
  if (m.scale() == GATED_VARIANCE) u = mul2(u, scale_pair(rest2_pair(d.a, d.rest)));
  return Run{d.a, u};
}
// Backward: its factor, what comes in from above, and what dx and di have per unit of G, df and drate per unit of a G
struct GatedBack { uint64_t a, up, dx, di, df, drate; };
// h: the state in front of it, and then behind; dz: the gradient of z
template <typename T, bool FAR, class M>
__device__ __forceinline__ GatedBack gated_token_bw(const M& m, uint64_t f, uint64_t x, uint64_t i, uint64_t z, uint64_t dy, uint64_t rate, uint64_t& h, uint64_t& dz) {
  GatedBack t;
  const Decay d = gated_decay<T, FAR, true>(m, f, rate);
  t.a = d.a;
  uint64_t gx = x, cg = 0, w = h, u;
  t.dx = dup2(1.f);
  if (m.i()) {
    logistic_both<T>(i, t.dx, cg);
    gx = mul2(t.dx, gx);
  }
  u = gx;
  if (m.scale() == GATED_CONVEX) {
    w = minus2(h, gx);
    u = mul2(gx, d.rest);
    t.dx = m.i() ? mul2(t.dx, d.rest) : d.rest;
  }
  if (m.scale() == GATED_VARIANCE) {
    const uint64_t q2 = rest2_pair(d.a, d.rest), inv = inv_scale_pair(q2), s = mul2(q2, inv);
    w = minus2(h, mul2(mul2(d.a, gx), inv));
    u = mul2(gx, s);
    t.dx = m.i() ? mul2(t.dx, s) : s;
  }
  t.di = m.i() ? mul2(u, cg) : 0;
  if (m.rate()) {
    t.drate = mul2(w, d.sf);
    t.df = mul2(mul2(t.drate, rate), d.cf);
  } else {
    t.drate = 0;
    t.df = mul2(w, d.rest);
  }
  h = fma2(d.a, h, u);
  t.up = dy;
  if (m.z()) {
    uint64_t s, c;
    logistic_both<T>(z, s, c);
    dz = mul2(mul2(dy, h), mul2(s, fma2(z, c, dup2(1.f))));
    t.up = mul2(dy, mul2(z, s));
  }
  return t;
}

// ---- channels in rows of 16 bytes ----------------------------------------------------------------------
// The operands come by asynchronous copies, a tile ahead: each warp copies its own rows (of its 32 lanes' V channels), so that only it
// waits for them.  Rows behind the sequence and channels behind the last are zeros.
constexpr int GATED_STAGES = 2;
template <typename T, int V> struct GatedRows {
  static constexpr int CH = 32 * V, BYTES = CH * (int)sizeof(T), CHUNKS = BYTES / 16, PER = 32 / CHUNKS, E = 16 / (int)sizeof(T);
  static_assert(CHUNKS <= 32 && GL % PER == 0, "");
  int row, col;   // of this lane's first chunk, and its channel
  bool ok;
  __device__ GatedRows(int first, int D) : row((threadIdx.x & 31) / CHUNKS), col(((threadIdx.x & 31) % CHUNKS) * E), ok(first + col < D) {}
  // x: this sequence, at the warp's first channel; tokens t0 ... t0 + 7 to dst[8][CH]
  __device__ __forceinline__ void copy(T* dst, const T* x, long long stride, int t0, int S) const {
    const T* src = x + (ok ? col : 0);
#pragma unroll
    for (int k = 0; k < GL; k += PER) {
      const int t = t0 + k + row;
      const bool in = ok && t < S;
      copy_async<T, E>(dst + (k + row) * CH + col, src + (in ? t : 0) * stride, in);
    }
  }
};
template <typename T, int V> __device__ __forceinline__ void get_pairs(const T* p, uint64_t (&o)[V / 2]) {
  const Pack<T, V> v = load_pack<T, V>(p);
#pragma unroll
  for (int k = 0; k < V / 2; ++k) o[k] = f2(to_f32(v.e[2 * k]), to_f32(v.e[2 * k + 1]));
}
template <typename T, int V> __device__ __forceinline__ void put_pairs(T* p, const uint64_t (&v)[V / 2]) {
  float o[V];
#pragma unroll
  for (int k = 0; k < V / 2; ++k) unf2(v[k], o[2 * k], o[2 * k + 1]);
  store_pack(p, pack<T, V>(o));
}

template <typename T, int V, class M> __global__ void __launch_bounds__(32 * GATED_WARPS, 2) gated_fw_rows(GatedPtrs<T> p, GatedDims q, M m) {
  constexpr int P = V / 2, CH = 32 * V, NT = 2 + M::i() + M::z(), ROWS = GL * CH;
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  GatedShared<P>& sh = *reinterpret_cast<GatedShared<P>*>(shared_bytes);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5, tile = W * GL;
  T* const tiles = reinterpret_cast<T*>(shared_bytes + sizeof(GatedShared<P>)) + warp * (GATED_STAGES * NT * ROWS);   // this warp's [stage][tensor][8][CH]
  auto fetch = [&](int unit, int stage) {
    if (unit < q.units) {
      const Unit u = unit_of(unit, q);
      T* const dst = tiles + stage * (NT * ROWS);
      const int t0 = u.k * tile + warp * GL, first = u.block * CH;
      const GatedRows<T, V> rows(first, q.D);
      rows.copy(dst, p.f + u.b * q.fb + first, q.ft, t0, q.S);
      rows.copy(dst + ROWS, p.x + u.b * q.xb + first, q.xt, t0, q.S);
      if (m.i()) rows.copy(dst + 2 * ROWS, p.i + u.b * q.ib + first, q.it, t0, q.S);
      if (m.z()) rows.copy(dst + (NT - 1) * ROWS, p.z + u.b * q.zb + first, q.zt, t0, q.S);
    }
    cp_commit();
  };
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < GATED_STAGES; ++s) sh.unit[s] = take_unit(q, s);
  }
  __syncthreads();
  int now = sh.unit[0], next = sh.unit[1];
  fetch(now, 0);
  fetch(next, 1);
  __syncthreads();   // the numbers have been read
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    const int t0 = u.k * tile + warp * GL, n = q.S - t0, ch = u.block * CH + lane * V, stage = turn % GATED_STAGES;
    const bool ok = ch < q.D;
    const T* const mine_x = tiles + stage * (NT * ROWS) + lane * V;
    int after = 0;
    if (threadIdx.x == 0) after = take_unit(q, turn + GATED_STAGES);
    uint64_t rate[P] = {}, first[P] = {};
    if (ok && m.rate()) get_pairs<float, V>(p.rate + ch, rate);
    if (ok && warp == 0 && u.k < q.group && p.h0 != nullptr) get_pairs<float, V>(p.h0 + (long long)u.b * q.D + ch, first);
    bool far = false;
    if (m.rate()) {
#pragma unroll
      for (int k = 0; k < P; ++k) far = far || far_rate(rate[k]);
      far = __any_sync(0xffffffffu, far);
    }
    Run r[GL][P];
    cp_wait<GATED_STAGES - 1>();
    __syncwarp();
    auto tokens = [&](auto far_) {
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        uint64_t f[P], x[P], i[P] = {};
        get_pairs<T, V>(mine_x + j * CH, f);
        get_pairs<T, V>(mine_x + ROWS + j * CH, x);
        if (m.i()) get_pairs<T, V>(mine_x + 2 * ROWS + j * CH, i);
#pragma unroll
        for (int k = 0; k < P; ++k) r[j][k] = gated_token<T, decltype(far_)::value>(m, f[k], x[k], i[k], rate[k]);
      }
    };
    if (m.rate() && far) tokens(std::true_type{});
    else tokens(std::false_type{});
    if (n < GL) {   // tokens behind the last leave the state as it is
#pragma unroll
      for (int j = 0; j < GL; ++j)
#pragma unroll
        for (int k = 0; k < P; ++k)
          if (j >= n) r[j][k] = no_tokens();
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      Run mine = r[0][k];
#pragma unroll
      for (int j = 1; j < GL; ++j) mine = then(mine, r[j][k]);
      sh.part[warp][k][lane] = mine;
    }
    if (threadIdx.x == 0) sh.unit[stage] = after;
    __syncthreads();
    after = sh.unit[stage];
    Run front[P];
    gated_front<false, P>(sh, front);
    if (warp == 0) {
      uint64_t end[P];
      gated_unit_start<false, P>(sh, q, u, first, end);
      if (p.h_last != nullptr && u.k == q.nt - 1 && ok) put_pairs<float, V>(p.h_last + (long long)u.b * q.D + ch, end);
    }
    if (!m.z()) fetch(after, stage);   // (this warp has read its rows)
    __syncthreads();
    if (n > 0) {
      uint64_t h[P];
#pragma unroll
      for (int k = 0; k < P; ++k) h[k] = through(front[k], sh.start[k][lane]);
      if (p.ckpt != nullptr && ok) put_pairs<float, V>(p.ckpt + ((long long)u.b * q.nc + t0 / GL) * q.D + ch, h);
      T* py = p.y + ((long long)u.b * q.S + t0) * q.D + ch;
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        uint64_t o[P], z[P] = {};
        if (m.z()) get_pairs<T, V>(mine_x + (NT - 1) * ROWS + j * CH, z);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          h[k] = through(r[j][k], h[k]);
          o[k] = m.z() ? mul2(h[k], mul2(z[k], logistic_pair2<T>(z[k]))) : h[k];
        }
        if (ok && j < n) put_pairs<T, V>(py, o);
        py += q.D;
      }
    }
    if (m.z()) {
      __syncwarp();
      fetch(after, stage);
    }
    now = next;
    next = after;
  }
}

// Sums of drate over a unit's warps, in order, by its last warp
__device__ __forceinline__ uint64_t gated_rate_of(const uint64_t (&sums)[GATED_WARPS][32]) {
  uint64_t s = sums[0][threadIdx.x & 31];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) s = add2(s, sums[w][threadIdx.x & 31]);
  return s;
}

template <typename T, class M> __global__ void __launch_bounds__(32 * GATED_WARPS, 2) gated_bw_rows(GatedPtrs<T> p, GatedDims q, M m) {
  constexpr int V = 2, CH = 32 * V, NT = 3 + M::i() + M::z(), ROWS = GL * CH;
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  GatedShared<1>& sh = *reinterpret_cast<GatedShared<1>*>(shared_bytes);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5, tile = W * GL;
  T* const tiles = reinterpret_cast<T*>(shared_bytes + sizeof(GatedShared<1>)) + warp * (GATED_STAGES * NT * ROWS);
  auto fetch = [&](int unit, int stage) {
    if (unit < q.units) {
      const Unit u = unit_of(unit, q);
      T* const dst = tiles + stage * (NT * ROWS);
      const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, first = u.block * CH;   // the last tokens first
      const GatedRows<T, V> rows(first, q.D);
      rows.copy(dst, p.f + u.b * q.fb + first, q.ft, t0, q.S);
      rows.copy(dst + ROWS, p.x + u.b * q.xb + first, q.xt, t0, q.S);
      rows.copy(dst + 2 * ROWS, p.dy + u.b * q.gb + first, q.gt, t0, q.S);
      if (m.i()) rows.copy(dst + 3 * ROWS, p.i + u.b * q.ib + first, q.it, t0, q.S);
      if (m.z()) rows.copy(dst + (NT - 1) * ROWS, p.z + u.b * q.zb + first, q.zt, t0, q.S);
    }
    cp_commit();
  };
  auto state = [&](int unit) {   // in front of this thread's run
    uint64_t h[1] = {0};
    if (unit < q.units) {
      const Unit u = unit_of(unit, q);
      const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, ch = u.block * CH + lane * V;
      if (t0 < q.S && ch < q.D) get_pairs<float, 2>(p.ckpt_in + ((long long)u.b * q.nc + t0 / GL) * q.D + ch, h);
    }
    return h[0];
  };
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < GATED_STAGES; ++s) sh.unit[s] = take_unit(q, s);
  }
  __syncthreads();
  int now = sh.unit[0], next = sh.unit[1];
  fetch(now, 0);
  fetch(next, 1);
  uint64_t h_next = state(now);
  float* rate_to = nullptr;   // where the sums of the unit before go
  __syncthreads();
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, n = q.S - t0, ch = u.block * CH + lane * V, stage = turn % GATED_STAGES;
    const bool ok = ch < q.D;
    const T* const mine_x = tiles + stage * (NT * ROWS) + lane * V;
    const long long at = ((long long)u.b * q.S + t0) * q.D + ch;
    int after = 0;
    if (threadIdx.x == 0) after = take_unit(q, turn + GATED_STAGES);
    uint64_t rate[1] = {0}, first[1] = {0}, drate = 0, h = h_next;
    if (ok && m.rate()) get_pairs<float, 2>(p.rate + ch, rate);
    if (ok && warp == 0 && u.k < q.group && p.dh_last != nullptr) get_pairs<float, 2>(p.dh_last + (long long)u.b * q.D + ch, first);
    const bool far = m.rate() && __any_sync(0xffffffffu, far_rate(rate[0]));
    GatedBack k[GL];
    cp_wait<GATED_STAGES - 1>();
    __syncwarp();
    auto tokens = [&](auto far_) {
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        auto get = [&](int tensor) {
          uint64_t v[1];
          get_pairs<T, 2>(mine_x + tensor * ROWS + j * CH, v);
          return v[0];
        };
        uint64_t dz[1];
        k[j] = gated_token_bw<T, decltype(far_)::value>(m, get(0), get(1), m.i() ? get(3) : 0, m.z() ? get(NT - 1) : 0, get(2), rate[0], h, dz[0]);
        if (m.z() && ok && j < n) put_pairs<T, 2>(p.dz + at + (long long)j * q.D, dz);
      }
    };
    if (far) tokens(std::true_type{});
    else tokens(std::false_type{});
    if (n < GL) {
#pragma unroll
      for (int j = 0; j < GL; ++j)
        if (j >= n) k[j].a = dup2(1.f), k[j].up = 0;
    }
    Run mine = no_tokens();
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) mine = Run{mul2(k[j].a, mine.A), mul2(k[j].a, add2(k[j].up, mine.H))};
    sh.part[warp][0][lane] = mine;
    if (threadIdx.x == 0) sh.unit[stage] = after;
    __syncthreads();
    after = sh.unit[stage];
    h_next = state(next);
    Run front[1];
    gated_front<true, 1>(sh, front);
    if (warp == 0) {
      uint64_t end[1];
      gated_unit_start<true, 1>(sh, q, u, first, end);
      if (p.dh0 != nullptr && u.k == q.nt - 1 && ok) put_pairs<float, 2>(p.dh0 + (long long)u.b * q.D + ch, end);
    }
    if (m.rate() && warp == W - 1 && rate_to != nullptr) {
      const uint64_t o[1] = {gated_rate_of(sh.drate)};
      put_pairs<float, 2>(rate_to, o);
    }
    fetch(after, stage);
    __syncthreads();
    if (n > 0) {
      uint64_t c = through(front[0], sh.start[0][lane]);
#pragma unroll
      for (int j = GL - 1; j >= 0; --j) {
        const uint64_t G = add2(k[j].up, c);
        c = mul2(k[j].a, G);
        if (j >= n) continue;
        if (m.rate()) drate = fma2(c, k[j].drate, drate);
        const uint64_t dx[1] = {mul2(G, k[j].dx)}, df[1] = {mul2(c, k[j].df)}, di[1] = {mul2(G, k[j].di)};
        if (ok) put_pairs<T, 2>(p.dx + at + (long long)j * q.D, dx);
        if (ok) put_pairs<T, 2>(p.df + at + (long long)j * q.D, df);
        if (m.i() && ok) put_pairs<T, 2>(p.di + at + (long long)j * q.D, di);
      }
    }
    if (m.rate()) {
      sh.drate[warp][lane] = drate;
      rate_to = p.rate_parts != nullptr && ok ? p.rate_parts + ((long long)u.b * q.nt + u.k) * q.D + ch : nullptr;
    }
    now = next;
    next = after;
  }
  if (m.rate()) {
    __syncthreads();
    if (warp == W - 1 && rate_to != nullptr) {
      const uint64_t o[1] = {gated_rate_of(sh.drate)};
      put_pairs<float, 2>(rate_to, o);
    }
  }
}

// ---- channels one by one: any width, any alignment -----------------------------------------------------
template <typename T> __device__ __forceinline__ uint64_t one(const T* p) { return f2(to_f32(*p), 0.f); }
template <typename T> __device__ __forceinline__ void put_one(T* p, uint64_t v) {
  float lo, hi;
  unf2(v, lo, hi);
  *p = from_f32<T>(lo);
}

template <typename T> __global__ void __launch_bounds__(32 * GATED_WARPS, 2) gated_fw_any(GatedPtrs<T> p, GatedDims q, GatedAny m) {
  __shared__ GatedShared<1> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tile = (blockDim.x >> 5) * GL;
  for (int turn = 0;; ++turn) {
    if (threadIdx.x == 0) sh.unit[0] = take_unit(q, turn);
    __syncthreads();
    const int unit = sh.unit[0];
    if (unit >= q.units) return;
    const Unit u = unit_of(unit, q);
    const int t0 = u.k * tile + warp * GL, n = q.S - t0, own = u.block * 32 + lane, ch = min(own, q.D - 1);   // (n: may be none, or more)
    const bool ok = own < q.D;
    const uint64_t rate = m.rate() ? one(p.rate + ch) : 0, first[1] = {p.h0 != nullptr ? one(p.h0 + (long long)u.b * q.D + ch) : 0};
    Run r[GL], mine = no_tokens();
    T rx[GL], rf[GL], ri[GL];
    const T *px = p.x + u.b * q.xb + t0 * q.xt + ch, *pf = p.f + u.b * q.fb + t0 * q.ft + ch, *pi = m.i() ? p.i + u.b * q.ib + t0 * q.it + ch : nullptr;
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      if (j >= n) break;
      rf[j] = pf[j * q.ft];
      rx[j] = px[j * q.xt];
      if (m.i()) ri[j] = pi[j * q.it];
    }
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      r[j] = j < n ? gated_token<T, true>(m, one(rf + j), one(rx + j), m.i() ? one(ri + j) : 0, rate) : no_tokens();
      mine = then(mine, r[j]);
    }
    sh.part[warp][0][lane] = mine;
    __syncthreads();
    Run front[1];
    gated_front<false, 1>(sh, front);
    if (warp == 0) {
      uint64_t end[1];
      gated_unit_start<false, 1>(sh, q, u, first, end);
      if (p.h_last != nullptr && u.k == q.nt - 1 && ok) put_one(p.h_last + (long long)u.b * q.D + ch, end[0]);
    }
    __syncthreads();
    if (n <= 0) continue;
    uint64_t h = through(front[0], sh.start[0][lane]);
    if (p.ckpt != nullptr && ok) put_one(p.ckpt + ((long long)u.b * q.nc + t0 / GL) * q.D + ch, h);
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      if (j >= n) break;
      h = through(r[j], h);
      uint64_t o = h;
      if (m.z()) {
        const uint64_t z = one(p.z + u.b * q.zb + (t0 + j) * q.zt + ch);
        o = mul2(o, mul2(z, logistic_pair2<T>(z)));
      }
      if (ok) put_one(p.y + ((long long)u.b * q.S + t0 + j) * q.D + ch, o);
    }
  }
}

template <typename T> __global__ void __launch_bounds__(32 * GATED_WARPS) gated_bw_any(GatedPtrs<T> p, GatedDims q, GatedAny m) {
  __shared__ GatedShared<1> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5, tile = W * GL;
  for (int turn = 0;; ++turn) {
    if (threadIdx.x == 0) sh.unit[0] = take_unit(q, turn);
    __syncthreads();
    const int unit = sh.unit[0];
    if (unit >= q.units) return;
    const Unit u = unit_of(unit, q);
    const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, n = q.S - t0, own = u.block * 32 + lane, ch = min(own, q.D - 1);
    const bool ok = own < q.D;
    const uint64_t rate = m.rate() ? one(p.rate + ch) : 0, first[1] = {p.dh_last != nullptr ? one(p.dh_last + (long long)u.b * q.D + ch) : 0};
    const long long at = ((long long)u.b * q.S + t0) * q.D + ch;
    uint64_t drate = 0;
    GatedBack k[GL];
    T rx[GL], rf[GL], ri[GL], rz[GL], rg[GL];
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      if (j >= n) break;
      rf[j] = p.f[u.b * q.fb + (t0 + j) * q.ft + ch];
      rx[j] = p.x[u.b * q.xb + (t0 + j) * q.xt + ch];
      rg[j] = p.dy[u.b * q.gb + (t0 + j) * q.gt + ch];
      if (m.i()) ri[j] = p.i[u.b * q.ib + (t0 + j) * q.it + ch];
      if (m.z()) rz[j] = p.z[u.b * q.zb + (t0 + j) * q.zt + ch];
    }
    uint64_t h = n > 0 ? one(p.ckpt_in + ((long long)u.b * q.nc + t0 / GL) * q.D + ch) : 0;
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      k[j].a = dup2(1.f), k[j].up = 0;
      if (j >= n) continue;
      uint64_t dz = 0;
      k[j] = gated_token_bw<T, true>(m, one(rf + j), one(rx + j), m.i() ? one(ri + j) : 0, m.z() ? one(rz + j) : 0, one(rg + j), rate, h, dz);
      if (m.z() && ok) put_one(p.dz + at + (long long)j * q.D, dz);
    }
    Run mine = no_tokens();
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) mine = Run{mul2(k[j].a, mine.A), mul2(k[j].a, add2(k[j].up, mine.H))};
    sh.part[warp][0][lane] = mine;
    __syncthreads();
    Run front[1];
    gated_front<true, 1>(sh, front);
    if (warp == 0) {
      uint64_t end[1];
      gated_unit_start<true, 1>(sh, q, u, first, end);
      if (p.dh0 != nullptr && u.k == q.nt - 1 && ok) put_one(p.dh0 + (long long)u.b * q.D + ch, end[0]);
    }
    __syncthreads();
    uint64_t c = through(front[0], sh.start[0][lane]);
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) {
      if (j >= n) continue;
      const uint64_t G = add2(k[j].up, c);
      c = mul2(k[j].a, G);
      if (m.rate()) drate = fma2(c, k[j].drate, drate);
      if (ok) put_one(p.dx + at + (long long)j * q.D, mul2(G, k[j].dx));
      if (ok) put_one(p.df + at + (long long)j * q.D, mul2(c, k[j].df));
      if (m.i() && ok) put_one(p.di + at + (long long)j * q.D, mul2(G, k[j].di));
    }
    if (m.rate() && p.rate_parts != nullptr) {
      sh.drate[warp][lane] = drate;
      __syncthreads();
      if (warp == W - 1 && ok) put_one(p.rate_parts + ((long long)u.b * q.nt + u.k) * q.D + ch, gated_rate_of(sh.drate));
    }
  }
}

// ---- launches -----------------------------------------------------------------------------------------
template <typename T, class M> int gated_launch(void (*kern)(GatedPtrs<T>, GatedDims, M), size_t smem, const GatedPtrs<T>& p, const GatedDims& q, M m,
                                                cudaStream_t st) {
  if (smem > 48 * 1024) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  int held = 0;
  MLSTM_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kern, 32 * q.warps, smem));
  const long long grid = std::min((long long)q.units, (long long)std::max(held, 1) * sm_count());
  kern<<<(unsigned)grid, 32 * q.warps, smem, st>>>(p, q, m);
  MLSTM_LAUNCH_CHECK();
  return MLSTM_OK;
}

template <typename T> int gated_run(bool back, int V, const GatedPtrs<T>& p, const GatedDims& q, cudaStream_t st) {
  constexpr int FV = 8 / (int)sizeof(T);
  const bool rate = p.rate != nullptr, i = p.i != nullptr, z = p.z != nullptr;
  if (V == 1) return gated_launch<T, GatedAny>(back ? gated_bw_any<T> : gated_fw_any<T>, 0, p, q, GatedAny{rate, i, z, q.scale}, st);
  const size_t rows = (size_t)q.warps * GATED_STAGES * GL * 32 * sizeof(T) * (2 + back + i + z);
  auto pick = [&](auto r, auto s, auto ii, auto zz) {
    using M = GatedFixed<decltype(r)::value, decltype(s)::value, decltype(ii)::value, decltype(zz)::value>;
    if (back) return gated_launch<T, M>(gated_bw_rows<T, M>, rows * 2 + sizeof(GatedShared<1>), p, q, M{}, st);
    return gated_launch<T, M>(gated_fw_rows<T, FV, M>, rows * FV + sizeof(GatedShared<FV / 2>), p, q, M{}, st);
  };
  auto with_z = [&](auto r, auto s, auto ii) { return z ? pick(r, s, ii, std::true_type{}) : pick(r, s, ii, std::false_type{}); };
  auto with_i = [&](auto r, auto s) { return i ? with_z(r, s, std::true_type{}) : with_z(r, s, std::false_type{}); };
  auto with_scale = [&](auto r) {
    return q.scale == GATED_PLAIN    ? with_i(r, std::integral_constant<int, GATED_PLAIN>{})
           : q.scale == GATED_CONVEX ? with_i(r, std::integral_constant<int, GATED_CONVEX>{})
                                     : with_i(r, std::integral_constant<int, GATED_VARIANCE>{});
  };
  return rate ? with_scale(std::true_type{}) : with_scale(std::false_type{});
}
static int gated_status_of(int reset, int* status) {
  MLSTM_CUDA_CHECK(cudaMemcpyFromSymbol(status, g_gated_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    MLSTM_CUDA_CHECK(cudaMemcpyToSymbol(g_gated_status, &zero, sizeof(int)));
  }
  return MLSTM_OK;
}

}  // namespace mlstm
