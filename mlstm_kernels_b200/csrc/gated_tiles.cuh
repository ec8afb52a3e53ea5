// Gated linear recurrence over sequences: forward and backward kernels of one element type (formulas: gated.cuh).
//
// A run of tokens acts on the state before it as h -> A h + H (A the product of its factors, H its own end state), and two runs after
// one another as A2 A1, A2 H1 + H2.  A thread takes GATED_CK tokens of two channels in registers, the warps of a CTA take runs that
// follow one another: a unit (gated_units.h).  One pass over the data: every thread reduces its run to (A, H), the CTA's last warp, which
// takes no tokens, works out the state in front of every run, and every thread takes its tokens again out of its registers.
//
// Between units the states go through global memory.  CTAs take units in the order of their numbers, by a counter; what a unit waits
// for has a lower number, so that a CTA that runs has it or has done it: no unit waits for one that is not under way.  A unit
// publishes its own (A, H) as soon as it has it; the state in front of a group of units is published by the last unit of the group
// before.  A unit joins the runs of its group in front of it, always in that order, and takes the state in front of the group through
// them: results do not depend on who ran when.  The last warp looks for these while the others work on their tokens; how often it looks
// is bounded.  A value in global memory says by itself that it is there: the scratch is zero before, and +0 is published as -0, so
// that neither fences nor flags stand between two CTAs.
//
// The backward is the same in the other direction, on a_t (dyh_t + .): the forward has kept the state in front of every run, so that
// the states are recomputed without an exchange.
//
// What bounds it: waiting.  8 x 4096 x 2048 (bf16, i, rate, "variance") takes 163 us forward (3.5 TB/s) and 228 backward (4.3), where memory
// alone would take 87 and 149.  No unit is busy for the whole time: 54 and 55 % of the issue slots are used (about 90 and 135 instructions for 64
// elements), 55 and 38 % of the special functions' cycles; each of these is about half of the forward's time, and they overlap.  Of
// the resident warps' time 48 % forward and 30 % backward go to the two barriers of a unit: its warps keep their tokens in registers
// until the states in front of them come, and have nothing else to do meanwhile.  With few chains the states take longer: 1 x
// 65536 x 2048, twice the elements with 14 units of a chain under way at once, takes 505-560 us, 59 % of it at barriers (at 16384 tokens).
// Tokens held in shared memory instead (of an SM's 228 KB three CTAs with i use 156 forward, two 133 backward) would let a CTA reduce its
// next unit before the states of this one are there; that has not been built.
//
// Measured beside it, us forward / backward at 8 x 4096 x 2048: CTAs of a cluster that exchange runs through distributed shared memory
// 207-248 / 275-513; flags with fences 215 / 360; no warp of its own for the states, eight that take tokens, 283 / 395 (spills); one barrier
// a unit 160-173 / 300 (spills); two units at once in registers 172; four CTAs of 64 registers 179; three or five warps for tokens 189 / 335,
// 180 / 280.
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
constexpr int GL = GATED_CK;

// ---- units --------------------------------------------------------------------------------------------
// Code of the first wait that ran out since it was last asked for (0: none), read by the host
static __device__ int g_gated_status = 0;

__device__ __forceinline__ uint2 look(const uint2* p) {
  uint2 v;
  asm volatile("ld.relaxed.gpu.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 look(const uint4* p) {
  uint4 v;
  asm volatile("ld.relaxed.gpu.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 published(uint64_t v) {
  uint2 o = make_uint2((unsigned)v, (unsigned)(v >> 32));
  o.x = o.x == 0 ? 0x80000000u : o.x;
  o.y = o.y == 0 ? 0x80000000u : o.y;
  return o;
}
__device__ __forceinline__ void publish(uint2* p, uint64_t v) {
  const uint2 o = published(v);
  asm volatile("st.relaxed.gpu.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(o.x), "r"(o.y) : "memory");
}
__device__ __forceinline__ void publish(uint4* p, Run r) {
  const uint2 a = published(r.A), h = published(r.H);
  asm volatile("st.relaxed.gpu.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(h.x), "r"(h.y) : "memory");
}
__device__ __forceinline__ uint64_t word(unsigned lo, unsigned hi) { return (uint64_t)hi << 32 | lo; }

struct Unit { int k, chain, b, block; };   // its place in the chain (BACK: from the end), and the chain's
__device__ __forceinline__ Unit unit_of(int u, const GatedDims& q) {
  Unit o;
  o.k = q.chains(u);
  o.chain = u - o.k * (int)q.chains.d;
  o.b = q.blocks(o.chain);
  o.block = o.chain - o.b * (int)q.blocks.d;
  return o;
}

// The state in front of a unit, by a whole warp, a pair of channels to a lane: look() until it is there.
struct GatedFind {
  const uint4* agg;      // the runs of the group's units
  const uint2* state;    // the state in front of the group
  int pos, n;            // runs in front of the unit, and how many of them have been joined
  bool have;
  Run front;
  uint64_t h;
  // first: the state in front of the unit's chain
  __device__ __forceinline__ GatedFind(const GatedDims& q, const Unit& u, uint64_t first) : n(0), front(no_tokens()), h(first) {
    const int lane = threadIdx.x & 31, group = u.k / q.group;
    pos = u.k - group * q.group;
    have = group == 0;
    agg = q.agg + ((long long)u.chain * q.nt + u.k - pos) * 32 + lane;
    state = q.state + ((long long)u.chain * q.groups + group) * 32 + lane;
  }
  __device__ __forceinline__ bool there() const { return have && n == pos; }
  __device__ __forceinline__ uint64_t value() const { return through(front, h); }
  __device__ __forceinline__ void look_again() {
    constexpr int AT_ONCE = 4;
    uint4 r[AT_ONCE];
    uint2 s = make_uint2(0, 0);
    if (!have) s = look(state);
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (n + k < pos) r[k] = look(agg + (n + k) * 32);
    if (!have && __all_sync(0xffffffffu, s.x != 0 && s.y != 0)) {
      have = true;
      h = word(s.x, s.y);
    }
    const int end = min(n + AT_ONCE, pos);
    bool all = true;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      if (!all || n >= end) continue;
      all = __all_sync(0xffffffffu, r[k].x != 0 && r[k].y != 0 && r[k].z != 0 && r[k].w != 0);
      if (all) {
        front = then(front, Run{word(r[k].x, r[k].y), word(r[k].z, r[k].w)});
        ++n;
      }
    }
  }
};

struct alignas(16) GatedShared {
  Run part[GATED_WARPS][32];             // the warps' runs
  uint64_t start[GATED_WARPS][32];       // the states in front of them
  uint64_t drate[2][GATED_WARPS][32];    // (backward) sums of a unit and the one before
  int unit[2];                           // units to come
  int runs;                              // how many warps' runs have been there, in all
};
// Two barriers between the warps that take tokens and the one that hands the states on: the runs are there; the states are there.
__device__ __forceinline__ void barrier_arrive(int id) { asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "r"(blockDim.x) : "memory"); }
__device__ __forceinline__ void barrier_wait(int id) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(blockDim.x) : "memory"); }
constexpr int RUNS_THERE = 1, STATES_THERE = 2;
// a warp's run is in place; `runs` lets the last warp see, without waiting, that the barrier has all of them
__device__ __forceinline__ void run_there(GatedShared& sh) {
  barrier_arrive(RUNS_THERE);
  if ((threadIdx.x & 31) == 0) atomicAdd(&sh.runs, 1);
}

// The next unit: by the counter, or, where no unit waits for another, every gridDim-th
__device__ __forceinline__ int take_unit(const GatedDims& q, int turn) {
  return q.ticket != nullptr ? (int)min(atomicAdd(q.ticket, 1u), 0x7fffffffu) : (int)min((long long)blockIdx.x + (long long)turn * gridDim.x, 0x7fffffffll);
}

// What the CTA's last warp does, from the first unit to the last.  first(u): the state in front of a chain; last(u, h): takes that
// behind it; sums(u): takes the sums of drate of a unit that is done.
template <bool BACK, class First, class Last, class Sums>
__device__ __forceinline__ void gated_hand_on(GatedShared& sh, const GatedDims& q, int now, int next, First first, Last last, Sums sums) {
  const int lane = threadIdx.x & 31, W = (blockDim.x >> 5) - 1;
  Unit before{};
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    int after = 0;
    if (lane == 0) after = take_unit(q, turn + 2);
    const int pos = u.k % q.group;
    const bool more = u.k < q.nt - 1, ends = pos == q.group - 1;
    GatedFind find(q, u, u.k < q.group ? first(u) : 0);
    auto give_run = [&] {
      Run all = sh.part[BACK ? W - 1 : 0][lane];
      for (int n = 1; n < W; ++n) all = then(all, sh.part[BACK ? W - 1 - n : n][lane]);
      publish(q.agg + ((long long)u.chain * q.nt + u.k) * 32 + lane, all);
    };
    bool runs = false, gave = !more || ends;   // its own run is wanted by the units of its group behind it
    unsigned looks = 0;
#pragma unroll 1
    while (!find.there()) {
      if (!runs && __any_sync(0xffffffffu, *static_cast<volatile int*>(&sh.runs) == W * (turn + 1))) {
        runs = true;
        barrier_wait(RUNS_THERE);
        if (!gave) give_run();   // as early as possible, unless the unit can go on itself
        gave = true;
      }
      find.look_again();
      // After q.looks of them, or once another wait of this launch has run out, it goes on without: the results are wrong, the
      // status says so, and every CTA ends.
      if (++looks % 256 == 0) {
        unsigned gone;
        asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(gone) : "l"(q.gave_up) : "memory");
        if (looks >= q.looks && lane == 0) {
          atomicExch(q.gave_up, 1u);
          atomicCAS(&g_gated_status, 0, 301);
        }
        if (__any_sync(0xffffffffu, gone != 0 || looks >= q.looks)) find.have = true, find.n = find.pos;
      }
    }
    uint64_t h = find.value();
    if (!runs) barrier_wait(RUNS_THERE);
    Run r[GATED_WARPS];
#pragma unroll
    for (int n = 0; n < GATED_WARPS; ++n)
      if (n < W) r[n] = sh.part[BACK ? W - 1 - n : n][lane];
#pragma unroll
    for (int n = 0; n < GATED_WARPS; ++n)
      if (n < W) {
        sh.start[BACK ? W - 1 - n : n][lane] = h;
        h = through(r[n], h);
      }
    if (lane == 0) sh.unit[turn & 1] = after;
    if (!gave) give_run();
    __syncwarp();
    barrier_arrive(STATES_THERE);
    if (more && ends) publish(q.state + ((long long)u.chain * q.groups + u.k / q.group + 1) * 32 + lane, h);
    if (!more) last(u, h);
    if (BACK && turn > 0) sums(before, (turn - 1) & 1);
    before = u;
    now = next;
    next = __shfl_sync(0xffffffffu, after, 0);
    if (BACK && now >= q.units) {   // the last unit's sums
      barrier_wait(RUNS_THERE);
      sums(before, turn & 1);
    }
  }
}

// ---- one token of a pair of channels, backward ----------------------------------------------------------
// Backward, what its run needs: its factor, and what comes in from above; what the gates' gradients need of f and z besides
struct GatedAbove { uint64_t a, up, rest, sf, cf, dz; };
template <typename T, bool FAR, class M> __device__ __forceinline__ GatedAbove gated_token_above(const M& m, uint64_t f, uint64_t z, uint64_t dy, uint64_t rate) {
  const Decay d = gated_decay<T, FAR, true>(m, f, rate);
  GatedAbove t{d.a, dy, d.rest, 0, 0, 0};
  if (m.rate()) t.sf = d.sf, t.cf = d.cf;
  if (m.z()) {
    uint64_t s, c;
    logistic_gate<T>(z, s, c);
    const uint64_t u = mul2(dy, s);
    t.up = mul2(u, z);
    t.dz = mul2(u, fma2(z, c, dup2(1.f)));
  }
  return t;
}
// Backward, what does not need G: what dx and di have per unit of G, df and drate per unit of a G
struct GatedBack { uint64_t dx, di, df, drate; };
// h: the state in front of it, and then behind
template <typename T, class M>
__device__ __forceinline__ GatedBack gated_token_bw(const M& m, const GatedAbove& d, uint64_t x, uint64_t i, uint64_t rate, uint64_t& h) {
  GatedBack t;
  uint64_t gx = x, cg = 0, w = h, u;
  t.dx = dup2(1.f);
  if (m.i()) {
    logistic_gate<T>(i, t.dx, cg);
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
  return t;
}

// ---- channels in rows of 16 bytes ----------------------------------------------------------------------
// The operands come by asynchronous copies, a unit ahead: each warp copies its own rows of 64 channels, so that only it waits for
// them.  Rows behind the sequence and channels behind the last are zeros.  Three CTAs of 80 registers a thread forward, two of 128
// backward.  (In f32 their operands leave room for two forward with one gate and one with both, and for one backward with any: 8 x 4096 x
// 2048 with i, rate and "variance" takes 211 us, 5.2 TB/s, and 354, 5.4.)  Whole runs go by 32-bit offsets from a base that the warp shares, and without bounds: 171 -> 164 us forward, 260 -> 240
// backward at 8 x 4096 x 2048; copies that pass L1 by 166 / 245.
constexpr int GATED_STAGES = 2;
template <typename T> struct GatedRows {
  static constexpr int CH = 64, CHUNKS = CH * (int)sizeof(T) / 16, PER = 32 / CHUNKS, E = 16 / (int)sizeof(T);   // copies of a row, rows of one instruction
  static_assert(GL % PER == 0, "");
  int row, col;   // of this lane's first copy, and its channel
  bool ok;
  __device__ GatedRows(int first, int D) : row((threadIdx.x & 31) / CHUNKS), col(((threadIdx.x & 31) % CHUNKS) * E), ok(first + col < D) {}
  // x: this sequence, at the first channel; tokens t0 ... t0 + 7 to dst[8][CH].  (Eight tokens are less than 2^31 bytes apart.)
  __device__ __forceinline__ void copy(T* dst, const T* x, long long stride, int t0, int S, bool whole) const {
    T* const to = dst + row * CH + col;
    if (whole) {
      const char* const base = reinterpret_cast<const char*>(x + t0 * stride);
      const unsigned step = (unsigned)stride * (unsigned)sizeof(T);
      unsigned at = row * step + col * (unsigned)sizeof(T);
#pragma unroll
      for (int k = 0; k < GL; k += PER) {
        copy_async<T, E>(to + k * CH, reinterpret_cast<const T*>(base + at), true);
        at += PER * step;
      }
    } else {
      const T* src = x + (ok ? col : 0);
#pragma unroll
      for (int k = 0; k < GL; k += PER) {
        const int t = t0 + k + row;
        const bool in = ok && t < S;
        copy_async<T, E>(to + k * CH, src + (in ? t : 0) * stride, in);
      }
    }
  }
};
// a value that is the same in the whole warp, which the compiler then knows
__device__ __forceinline__ int same(int v) { return __shfl_sync(0xffffffffu, v, 0); }
template <typename T> __device__ __forceinline__ uint64_t pair_of(const Pack<T, 2>& v) { return f2(to_f32(v.e[0]), to_f32(v.e[1])); }
template <typename T> __device__ __forceinline__ uint64_t get_pair(const T* p) { return pair_of(load_pack<T, 2>(p)); }
template <typename T> __device__ __forceinline__ void put_pair(T* p, uint64_t v) {
  float o[2];
  unf2(v, o[0], o[1]);
  store_pack(p, pack<T, 2>(o));
}
template <typename T> __device__ __forceinline__ void put_pair(T* row, unsigned at, uint64_t v) { put_pair(reinterpret_cast<T*>(reinterpret_cast<char*>(row) + at), v); }

template <typename T, class M> __global__ void __launch_bounds__(32 * (GATED_WARPS + 1), 3) gated_fw_rows(GatedPtrs<T> p, GatedDims q, M m) {
  constexpr int CH = 64, NT = 2 + M::i() + M::z(), ROWS = GL * CH;
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  GatedShared& sh = *reinterpret_cast<GatedShared*>(shared_bytes);
  const int lane = threadIdx.x & 31, warp = same(threadIdx.x >> 5), W = (blockDim.x >> 5) - 1, tile = W * GL;
  if (threadIdx.x == 0) sh.unit[0] = take_unit(q, 0), sh.unit[1] = take_unit(q, 1), sh.runs = 0;
  __syncthreads();
  int now = same(sh.unit[0]), next = same(sh.unit[1]);
  __syncthreads();   // (they have been read)
  if (warp == W) {
    gated_hand_on<false>(
        sh, q, now, next, [&](const Unit& u) { return p.h0 != nullptr && u.block * CH + 2 * lane < q.D ? get_pair(p.h0 + (long long)u.b * q.D + u.block * CH + 2 * lane) : 0; },
        [&](const Unit& u, uint64_t h) {
          if (p.h_last != nullptr && u.block * CH + 2 * lane < q.D) put_pair(p.h_last + (long long)u.b * q.D + u.block * CH + 2 * lane, h);
        },
        [](const Unit&, int) {});
    return;
  }
  T* const tiles = reinterpret_cast<T*>(shared_bytes + sizeof(GatedShared)) + warp * (GATED_STAGES * NT * ROWS);   // this warp's [stage][tensor][8][CH]
  auto fetch = [&](int unit, int stage) {
    if (unit < q.units) {
      const Unit u = unit_of(unit, q);
      T* const dst = tiles + stage * (NT * ROWS);
      const int t0 = u.k * tile + warp * GL, first = u.block * CH;
      const GatedRows<T> rows(first, q.D);
      const bool whole = t0 + GL <= q.S && first + CH <= q.D;
      rows.copy(dst, p.f + u.b * q.fb + first, q.ft, t0, q.S, whole);
      rows.copy(dst + ROWS, p.x + u.b * q.xb + first, q.xt, t0, q.S, whole);
      if (m.i()) rows.copy(dst + 2 * ROWS, p.i + u.b * q.ib + first, q.it, t0, q.S, whole);
      if (m.z()) rows.copy(dst + (NT - 1) * ROWS, p.z + u.b * q.zb + first, q.zt, t0, q.S, whole);
    }
    cp_commit();
  };
  fetch(now, 0);
  fetch(next, 1);
  auto rate_of = [&](int unit) {
    if (!m.rate() || unit >= q.units) return (uint64_t)0;
    const int ch = unit_of(unit, q).block * CH + lane * 2;
    return ch < q.D ? get_pair(p.rate + ch) : (uint64_t)0;
  };
  uint64_t rate_next = rate_of(now);
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    const int t0 = u.k * tile + warp * GL, n = q.S - t0, ch = u.block * CH + lane * 2, stage = turn % GATED_STAGES;
    const bool ok = ch < q.D;
    const T* const mine_x = tiles + stage * (NT * ROWS) + lane * 2;
    const uint64_t rate = rate_next;
    const bool far = m.rate() && __any_sync(0xffffffffu, far_rate(rate));
    Run r[GL];
    cp_wait<GATED_STAGES - 1>();
    __syncwarp();
    auto tokens = [&](auto far_) {
#pragma unroll
      for (int j = 0; j < GL; ++j)
        r[j] = gated_token<T, decltype(far_)::value>(m, get_pair(mine_x + j * CH), get_pair(mine_x + ROWS + j * CH),
                                                     m.i() ? get_pair(mine_x + 2 * ROWS + j * CH) : 0, rate);
    };
    if (far) tokens(std::true_type{});
    else tokens(std::false_type{});
    if (n < GL) {   // tokens behind the last leave the state as it is
#pragma unroll
      for (int j = 0; j < GL; ++j)
        if (j >= n) r[j] = no_tokens();
    }
    Run mine = r[0];
#pragma unroll
    for (int j = 1; j < GL; ++j) mine = then(mine, r[j]);
    sh.part[warp][lane] = mine;
    run_there(sh);
    rate_next = rate_of(next);
    barrier_wait(STATES_THERE);
    const int after = same(sh.unit[stage]);
    if (!m.z()) fetch(after, stage);
    uint64_t h = sh.start[warp][lane];
    auto finish = [&](auto whole) {
      T* const y = p.y + ((long long)u.b * q.S + t0) * q.D + u.block * CH;
      const unsigned step = (unsigned)q.D * (unsigned)sizeof(T);
      unsigned to = lane * 2 * (unsigned)sizeof(T);
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        if (!decltype(whole)::value && j >= n) break;
        h = through(r[j], h);
        uint64_t o = h;
        if (m.z()) {
          const uint64_t z = get_pair(mine_x + (NT - 1) * ROWS + j * CH);
          o = mul2(h, mul2(z, logistic_pair2<T>(z)));
        }
        put_pair(y, to, o);
        to += step;
      }
    };
    if (ok && n > 0) {
      if (p.ckpt != nullptr) put_pair(p.ckpt + ((long long)u.b * q.nc + t0 / GL) * q.D + u.block * CH, lane * 8, h);
      if (n >= GL) finish(std::true_type{});
      else finish(std::false_type{});
    }
    if (m.z()) {
      __syncwarp();
      fetch(after, stage);
    }
    now = next;
    next = after;
  }
}

template <typename T, class M> __global__ void __launch_bounds__(32 * (GATED_WARPS + 1), 2) gated_bw_rows(GatedPtrs<T> p, GatedDims q, M m) {
  constexpr int CH = 64, NT = 3 + M::i() + M::z(), ROWS = GL * CH;
  // The run is given away before the rest of the work on the tokens, which the search for the state in front of the unit goes beside.
  // (With a rate too much lies between the two for the registers: 240 -> 260 us at 8 x 4096 x 2048.)
  constexpr bool EARLY = !M::rate();
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  GatedShared& sh = *reinterpret_cast<GatedShared*>(shared_bytes);
  const int lane = threadIdx.x & 31, warp = same(threadIdx.x >> 5), W = (blockDim.x >> 5) - 1, tile = W * GL;
  if (threadIdx.x == 0) sh.unit[0] = take_unit(q, 0), sh.unit[1] = take_unit(q, 1), sh.runs = 0;
  __syncthreads();
  int now = same(sh.unit[0]), next = same(sh.unit[1]);
  __syncthreads();
  if (warp == W) {
    gated_hand_on<true>(
        sh, q, now, next,
        [&](const Unit& u) { return p.dh_last != nullptr && u.block * CH + 2 * lane < q.D ? get_pair(p.dh_last + (long long)u.b * q.D + u.block * CH + 2 * lane) : 0; },
        [&](const Unit& u, uint64_t h) {
          if (p.dh0 != nullptr && u.block * CH + 2 * lane < q.D) put_pair(p.dh0 + (long long)u.b * q.D + u.block * CH + 2 * lane, h);
        },
        [&](const Unit& u, int buf) {
          if (!m.rate() || p.rate_parts == nullptr) return;
          uint64_t s = sh.drate[buf][0][lane];   // over the warps, in order
          for (int w = 1; w < W; ++w) s = add2(s, sh.drate[buf][w][lane]);
          if (u.block * CH + 2 * lane < q.D) put_pair(p.rate_parts + ((long long)u.b * q.nt + u.k) * q.D + u.block * CH + 2 * lane, s);
        });
    return;
  }
  T* const tiles = reinterpret_cast<T*>(shared_bytes + sizeof(GatedShared)) + warp * (GATED_STAGES * NT * ROWS);
  auto fetch = [&](int unit, int stage) {
    if (unit < q.units) {
      const Unit u = unit_of(unit, q);
      T* const dst = tiles + stage * (NT * ROWS);
      const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, first = u.block * CH;   // the last tokens first
      const GatedRows<T> rows(first, q.D);
      const bool whole = t0 + GL <= q.S && first + CH <= q.D;
      rows.copy(dst, p.f + u.b * q.fb + first, q.ft, t0, q.S, whole);
      rows.copy(dst + ROWS, p.x + u.b * q.xb + first, q.xt, t0, q.S, whole);
      rows.copy(dst + 2 * ROWS, p.dy + u.b * q.gb + first, q.gt, t0, q.S, whole);
      if (m.i()) rows.copy(dst + 3 * ROWS, p.i + u.b * q.ib + first, q.it, t0, q.S, whole);
      if (m.z()) rows.copy(dst + (NT - 1) * ROWS, p.z + u.b * q.zb + first, q.zt, t0, q.S, whole);
    }
    cp_commit();
  };
  auto state = [&](int unit) {   // in front of this thread's run
    if (unit >= q.units) return (uint64_t)0;
    const Unit u = unit_of(unit, q);
    const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, ch = u.block * CH + lane * 2;
    return t0 < q.S && ch < q.D ? get_pair(p.ckpt_in + ((long long)u.b * q.nc + t0 / GL) * q.D + ch) : (uint64_t)0;
  };
  fetch(now, 0);
  fetch(next, 1);
  auto rate_of = [&](int unit) {
    if (!m.rate() || unit >= q.units) return (uint64_t)0;
    const int ch = unit_of(unit, q).block * CH + lane * 2;
    return ch < q.D ? get_pair(p.rate + ch) : (uint64_t)0;
  };
  uint64_t rate_next = rate_of(now);
  uint64_t h_next = state(now);
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, n = q.S - t0, ch = u.block * CH + lane * 2, stage = turn % GATED_STAGES;
    const bool ok = ch < q.D;
    const T* const mine_x = tiles + stage * (NT * ROWS) + lane * 2;
    const uint64_t rate = rate_next;
    const bool far = m.rate() && __any_sync(0xffffffffu, far_rate(rate));
    uint64_t h = h_next;
    GatedAbove d[GL];
    GatedBack k[GL];
    cp_wait<GATED_STAGES - 1>();
    __syncwarp();
    T* const dz_row = m.z() ? p.dz + ((long long)u.b * q.S + t0) * q.D + u.block * CH : nullptr;
    auto get = [&](int tensor, int j) { return get_pair(mine_x + tensor * ROWS + j * CH); };
    auto rest = [&](int j) {
      k[j] = gated_token_bw<T>(m, d[j], get(1, j), m.i() ? get(3, j) : 0, rate, h);
      if (m.z() && ok && j < n) put_pair(dz_row, lane * 2 * (unsigned)sizeof(T) + j * (unsigned)q.D * (unsigned)sizeof(T), mul2(d[j].dz, h));
    };
    auto tokens = [&](auto far_) {
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        d[j] = gated_token_above<T, decltype(far_)::value>(m, get(0, j), m.z() ? get(NT - 1, j) : 0, get(2, j), rate);
        if (!EARLY) rest(j);
      }
    };
    if (far) tokens(std::true_type{});
    else tokens(std::false_type{});
    if (n < GL) {
#pragma unroll
      for (int j = 0; j < GL; ++j)
        if (j >= n) d[j].a = dup2(1.f), d[j].up = 0;
    }
    Run mine = no_tokens();
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) mine = Run{mul2(d[j].a, mine.A), mul2(d[j].a, add2(d[j].up, mine.H))};
    sh.part[warp][lane] = mine;
    run_there(sh);
    if (EARLY) {
#pragma unroll
      for (int j = 0; j < GL; ++j) rest(j);
    }
    h_next = state(next);
    rate_next = rate_of(next);
    barrier_wait(STATES_THERE);
    const int after = same(sh.unit[stage]);
    fetch(after, stage);
    uint64_t c = sh.start[warp][lane], drate = 0;
    auto finish = [&](auto whole) {
      const long long at = ((long long)u.b * q.S + t0) * q.D + u.block * CH;
      T *const dx = p.dx + at, *const df = p.df + at, *const di = m.i() ? p.di + at : nullptr;
      const unsigned step = (unsigned)q.D * (unsigned)sizeof(T);
      unsigned to = lane * 2 * (unsigned)sizeof(T) + (GL - 1) * step;
#pragma unroll
      for (int j = GL - 1; j >= 0; --j) {
        if (decltype(whole)::value || j < n) {
          const uint64_t G = add2(d[j].up, c);
          c = mul2(d[j].a, G);
          if (m.rate()) drate = fma2(c, k[j].drate, drate);
          put_pair(dx, to, mul2(G, k[j].dx));
          put_pair(df, to, mul2(c, k[j].df));
          if (m.i()) put_pair(di, to, mul2(G, k[j].di));
        }
        to -= step;
      }
    };
    if (ok && n >= GL) finish(std::true_type{});
    else if (ok && n > 0) finish(std::false_type{});
    if (m.rate()) sh.drate[turn & 1][warp][lane] = drate;
    now = next;
    next = after;
    if (now >= q.units) barrier_arrive(RUNS_THERE);   // the last unit's sums
  }
}

// ---- channels one by one: any width, any alignment -----------------------------------------------------
// A lane's two channels are 32 apart, so that neighbouring lanes have neighbouring channels of any alignment.  Which gates there are is
// a number of the call here: there is one kernel of a type and direction.  4 x 4096 x 2049 (bf16) takes 154 us forward and 354 backward,
// 2048 channels in rows 102 and 132: two CTAs to an SM, and loads of single elements, a few of which are under way at once.
template <typename T> struct GatedApart {
  int c0, c1;        // where to read: the last channel for those behind it
  bool ok0, ok1;
  __device__ __forceinline__ GatedApart(const Unit& u, int D) {
    const int c = u.block * 64 + (threadIdx.x & 31);
    c0 = min(c, D - 1), c1 = min(c + 32, D - 1), ok0 = c < D, ok1 = c + 32 < D;
  }
  __device__ __forceinline__ Pack<T, 2> load(const T* row) const {
    Pack<T, 2> v;
    v.e[0] = row[c0], v.e[1] = row[c1];
    return v;
  }
  template <typename O> __device__ __forceinline__ void put(O* row, uint64_t v) const {
    float lo, hi;
    unf2(v, lo, hi);
    if (ok0) row[c0] = from_f32<O>(lo);
    if (ok1) row[c1] = from_f32<O>(hi);
  }
  __device__ __forceinline__ uint64_t get(const float* row) const { return f2(row[c0], row[c1]); }
};

template <typename T> __global__ void __launch_bounds__(32 * (GATED_WARPS + 1), 2) gated_fw_any(GatedPtrs<T> p, GatedDims q, GatedAny m) {
  __shared__ GatedShared sh;
  const int lane = threadIdx.x & 31, warp = same(threadIdx.x >> 5), W = (blockDim.x >> 5) - 1, tile = W * GL;
  if (threadIdx.x == 0) sh.unit[0] = take_unit(q, 0), sh.unit[1] = take_unit(q, 1), sh.runs = 0;
  __syncthreads();
  int now = same(sh.unit[0]), next = same(sh.unit[1]);
  __syncthreads();
  if (warp == W) {
    gated_hand_on<false>(
        sh, q, now, next, [&](const Unit& u) { return p.h0 != nullptr ? GatedApart<T>(u, q.D).get(p.h0 + (long long)u.b * q.D) : 0; },
        [&](const Unit& u, uint64_t h) {
          if (p.h_last != nullptr) GatedApart<T>(u, q.D).put(p.h_last + (long long)u.b * q.D, h);
        },
        [](const Unit&, int) {});
    return;
  }
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    const GatedApart<T> at(u, q.D);
    const int t0 = u.k * tile + warp * GL, n = q.S - t0;   // (n: may be none, or more)
    const uint64_t rate = m.rate() ? at.get(p.rate) : 0;
    Run r[GL], mine = no_tokens();
    Pack<T, 2> rx[GL], rf[GL], ri[GL], rz[GL];
    const T *pz = m.z() ? p.z + u.b * q.zb + t0 * q.zt : nullptr;
    const T *px = p.x + u.b * q.xb + t0 * q.xt, *pf = p.f + u.b * q.fb + t0 * q.ft, *pi = m.i() ? p.i + u.b * q.ib + t0 * q.it : nullptr;
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      if (j >= n) break;
      rf[j] = at.load(pf + j * q.ft);
      rx[j] = at.load(px + j * q.xt);
      if (m.i()) ri[j] = at.load(pi + j * q.it);
      if (m.z()) rz[j] = at.load(pz + j * q.zt);
    }
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      r[j] = j < n ? gated_token<T, true>(m, pair_of(rf[j]), pair_of(rx[j]), m.i() ? pair_of(ri[j]) : 0, rate) : no_tokens();
      mine = then(mine, r[j]);
    }
    sh.part[warp][lane] = mine;
    run_there(sh);
    barrier_wait(STATES_THERE);
    const int after = same(sh.unit[turn & 1]);
    uint64_t h = sh.start[warp][lane];
    if (n > 0 && p.ckpt != nullptr) at.put(p.ckpt + ((long long)u.b * q.nc + t0 / GL) * q.D, h);
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      if (j >= n) break;
      h = through(r[j], h);
      uint64_t o = h;
      if (m.z()) {
        const uint64_t z = pair_of(rz[j]);
        o = mul2(o, mul2(z, logistic_pair2<T>(z)));
      }
      at.put(p.y + ((long long)u.b * q.S + t0 + j) * q.D, o);
    }
    __syncwarp();
    now = next;
    next = after;
  }
}

template <typename T> __global__ void __launch_bounds__(32 * (GATED_WARPS + 1), 2) gated_bw_any(GatedPtrs<T> p, GatedDims q, GatedAny m) {
  __shared__ GatedShared sh;
  const int lane = threadIdx.x & 31, warp = same(threadIdx.x >> 5), W = (blockDim.x >> 5) - 1, tile = W * GL;
  if (threadIdx.x == 0) sh.unit[0] = take_unit(q, 0), sh.unit[1] = take_unit(q, 1), sh.runs = 0;
  __syncthreads();
  int now = same(sh.unit[0]), next = same(sh.unit[1]);
  __syncthreads();
  if (warp == W) {
    gated_hand_on<true>(
        sh, q, now, next, [&](const Unit& u) { return p.dh_last != nullptr ? GatedApart<T>(u, q.D).get(p.dh_last + (long long)u.b * q.D) : 0; },
        [&](const Unit& u, uint64_t h) {
          if (p.dh0 != nullptr) GatedApart<T>(u, q.D).put(p.dh0 + (long long)u.b * q.D, h);
        },
        [&](const Unit& u, int buf) {
          if (p.rate_parts == nullptr) return;
          uint64_t s = sh.drate[buf][0][lane];
          for (int w = 1; w < W; ++w) s = add2(s, sh.drate[buf][w][lane]);
          GatedApart<T>(u, q.D).put(p.rate_parts + ((long long)u.b * q.nt + u.k) * q.D, s);
        });
    return;
  }
  for (int turn = 0; now < q.units; ++turn) {
    const Unit u = unit_of(now, q);
    const GatedApart<T> at(u, q.D);
    const int t0 = (q.nt - 1 - u.k) * tile + warp * GL, n = q.S - t0;
    const uint64_t rate = m.rate() ? at.get(p.rate) : 0;
    const long long row = ((long long)u.b * q.S + t0) * q.D;
    uint64_t a[GL], up[GL];
    GatedBack k[GL];
    uint64_t h = n > 0 ? at.get(p.ckpt_in + ((long long)u.b * q.nc + t0 / GL) * q.D) : 0;
    constexpr int AT_ONCE = 2;   // tokens: with 4 and 8, 90 and 50 us more at 4 x 4096 x 2049 (registers)
#pragma unroll
    for (int j0 = 0; j0 < GL; j0 += AT_ONCE) {
      Pack<T, 2> rx[AT_ONCE], rf[AT_ONCE], ri[AT_ONCE], rz[AT_ONCE], rg[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int t = t0 + j0 + e;
        if (j0 + e >= n) break;
        rf[e] = at.load(p.f + u.b * q.fb + t * q.ft);
        rx[e] = at.load(p.x + u.b * q.xb + t * q.xt);
        rg[e] = at.load(p.dy + u.b * q.gb + t * q.gt);
        if (m.i()) ri[e] = at.load(p.i + u.b * q.ib + t * q.it);
        if (m.z()) rz[e] = at.load(p.z + u.b * q.zb + t * q.zt);
      }
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int j = j0 + e;
        a[j] = dup2(1.f), up[j] = 0;
        if (j >= n) continue;
        const GatedAbove d = gated_token_above<T, true>(m, pair_of(rf[e]), m.z() ? pair_of(rz[e]) : 0, pair_of(rg[e]), rate);
        a[j] = d.a, up[j] = d.up;
        k[j] = gated_token_bw<T>(m, d, pair_of(rx[e]), m.i() ? pair_of(ri[e]) : 0, rate, h);
        if (m.z()) at.put(p.dz + row + (long long)j * q.D, mul2(d.dz, h));
      }
    }
    Run mine = no_tokens();
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) mine = Run{mul2(a[j], mine.A), mul2(a[j], add2(up[j], mine.H))};
    __syncwarp();
    sh.part[warp][lane] = mine;
    run_there(sh);
    barrier_wait(STATES_THERE);
    const int after = same(sh.unit[turn & 1]);
    uint64_t c = sh.start[warp][lane], drate = 0;
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) {
      if (j >= n) continue;
      const uint64_t G = add2(up[j], c);
      c = mul2(a[j], G);
      if (m.rate()) drate = fma2(c, k[j].drate, drate);
      at.put(p.dx + row + (long long)j * q.D, mul2(G, k[j].dx));
      at.put(p.df + row + (long long)j * q.D, mul2(c, k[j].df));
      if (m.i()) at.put(p.di + row + (long long)j * q.D, mul2(G, k[j].di));
    }
    __syncwarp();
    if (m.rate()) sh.drate[turn & 1][warp][lane] = drate;
    now = next;
    next = after;
    if (now >= q.units) barrier_arrive(RUNS_THERE);   // the last unit's sums
  }
}

// ---- launches -----------------------------------------------------------------------------------------
template <typename T, class M> int gated_launch(void (*kern)(GatedPtrs<T>, GatedDims, M), size_t smem, const GatedPtrs<T>& p, const GatedDims& q, M m,
                                                cudaStream_t st) {
  if (int rc = allow_smem((const void*)kern, smem)) return rc;
  int held = 0;
  MLSTM_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kern, 32 * (q.warps + 1), smem));
  const long long grid = std::min((long long)q.units, (long long)std::max(held, 1) * sm_count());
  kern<<<(unsigned)grid, 32 * (q.warps + 1), smem, st>>>(p, q, m);
  MLSTM_LAUNCH_CHECK();
  return MLSTM_OK;
}

template <typename T> int gated_run(bool back, bool rows, const GatedPtrs<T>& p, const GatedDims& q, cudaStream_t st) {
  const bool rate = p.rate != nullptr, i = p.i != nullptr, z = p.z != nullptr;
  if (!rows) return gated_launch<T, GatedAny>(back ? gated_bw_any<T> : gated_fw_any<T>, 0, p, q, GatedAny{rate, i, z, q.scale}, st);
  const size_t smem = sizeof(GatedShared) + (size_t)q.warps * GATED_STAGES * GL * 64 * sizeof(T) * (2 + back + i + z);
  auto pick = [&](auto r, auto s, auto ii, auto zz) {
    using M = GatedFixed<decltype(r)::value, decltype(s)::value, decltype(ii)::value, decltype(zz)::value>;
    return gated_launch<T, M>(back ? gated_bw_rows<T, M> : gated_fw_rows<T, M>, smem, p, q, M{}, st);
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
