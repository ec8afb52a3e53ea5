// Gated linear recurrence over sequences: forward and backward kernels of one element type (formulas: gated.cuh).
//
// A run of tokens acts on the state before it as h -> A h + H (A the product of its factors, H its own end state), and two runs after
// one another as A2 A1, A2 H1 + H2.  A thread takes GATED_CK tokens of a pair of channels in registers; the warps of a CTA take runs
// that follow one another, and the CTAs of a cluster the CTAs' runs.  One pass over the data: every thread reduces its run to (A, H),
// these are exchanged in shared memory (within a cluster in every CTA's, written there by the others), every thread works out the
// state in front of its run from those before it, always in the same order, and then takes its tokens again out of its registers.
// Then all go on to the next tile of tokens.  The backward is the same in the other direction, on a_t (dyh_t + .): the
// forward has kept the state in front of every run, so that the states are recomputed without an exchange.
#pragma once
#include "gated.cuh"

namespace mlstm {

// What is there, known when a kernel is compiled, or when it is called (for channels that come one by one)
template <bool RATE, int SCALE, bool I, bool Z> struct GatedFixed {
  __device__ static constexpr bool rate() { return RATE; }
  __device__ static constexpr int scale() { return SCALE; }
  __device__ static constexpr bool i() { return I; }
  __device__ static constexpr bool z() { return Z; }
};
struct GatedAny {
  bool rate_, i_, z_;
  int scale_;
  __device__ bool rate() const { return rate_; }
  __device__ int scale() const { return scale_; }
  __device__ bool i() const { return i_; }
  __device__ bool z() const { return z_; }
};

template <typename T> struct GatedPtrs {
  const T *x, *f, *i, *z, *dy;
  const float *rate, *h0, *ckpt_in, *dh_last;
  T *y, *dx, *df, *di, *dz;
  float *h_last, *ckpt, *dh0, *rate_parts;
};

constexpr int GATED_WARPS = 8, GATED_CLUSTER = 16;
constexpr int GL = GATED_CK;

template <typename T, int V> __device__ __forceinline__ uint64_t pair_of(const Pack<T, V>& p) {
  if constexpr (V == 2) return f2(to_f32(p.e[0]), to_f32(p.e[1]));
  else return f2(to_f32(p.e[0]), 0.f);
}
template <typename T, int V> __device__ __forceinline__ void put_pair(T* p, uint64_t v) {
  float o[2];
  unf2(v, o[0], o[1]);
  if constexpr (V == 2) store_pack<T, 2>(p, pack<T, 2>(o));
  else *p = from_f32<T>(o[0]);
}
template <int V> __device__ __forceinline__ uint64_t get_f32(const float* p) {
  if constexpr (V == 2) return pair_of<float, 2>(load_pack<float, 2>(p));
  else return f2(*p, 0.f);
}

struct Run { uint64_t A, H; };
__device__ __forceinline__ Run no_tokens() { return Run{dup2(1.f), 0}; }
__device__ __forceinline__ Run then(Run first, Run second) { return Run{mul2(second.A, first.A), fma2(second.A, first.H, second.H)}; }
__device__ __forceinline__ uint64_t through(Run r, uint64_t h) { return fma2(r.A, h, r.H); }

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void put_remote(const Run* here, unsigned rank, Run v) {
  unsigned a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(here)), "r"(rank));
  asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(a), "l"(v.A), "l"(v.H) : "memory");
}

struct GatedShared {
  Run part[2][GATED_WARPS][32];
  Run total[2][GATED_CLUSTER][32];
};

// The state in front of this thread's run, of all runs in the cluster one after the other (BACK: from the last); `carry` goes from in
// front of the tile to behind it.  One barrier a tile: the buffers are two, taken in turn.
template <bool BACK> __device__ __forceinline__ uint64_t gated_exchange(GatedShared& sh, Run mine, uint64_t& carry, int buf, int K, int rank) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  __syncwarp();
  sh.part[buf][warp][lane] = mine;
  __syncthreads();
  uint64_t before = carry;
  if (K == 1) {
    for (int k = 0; k < W; ++k) {
      const int w = BACK ? W - 1 - k : k;
      if (w == warp) before = carry;
      carry = through(sh.part[buf][w][lane], carry);
    }
  } else {
    Run all = no_tokens(), front = no_tokens();
    for (int k = 0; k < W; ++k) {
      const int w = BACK ? W - 1 - k : k;
      if (w == warp) front = all;
      all = then(all, sh.part[buf][w][lane]);
    }
    for (int k = warp; k < K; k += W) put_remote(&sh.total[buf][rank][lane], k, all);
    cluster_sync_all();
    for (int k = 0; k < K; ++k) {
      const int c = BACK ? K - 1 - k : k;
      if (c == rank) before = through(front, carry);
      carry = through(sh.total[buf][c][lane], carry);
    }
  }
  return before;
}

// FAR: the rate may be outside (-1/2, 0]
template <typename T, bool FAR, class M> __device__ __forceinline__ Decay gated_decay(const M& m, uint64_t f, uint64_t rate) {
  if (m.rate()) return decay_pair<T, true, FAR>(f, rate);
  return decay_pair<T, false>(f, rate);
}

template <typename T, int V, class M> __global__ void __launch_bounds__(32 * GATED_WARPS) gated_fw(GatedPtrs<T> p, GatedDims q, M m) {
  __shared__ GatedShared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  const int K = q.K, rank = K > 1 ? (int)cluster_rank() : 0;
  const long long chain = blockIdx.x / K;
  const int b = (int)(chain / q.blocks), own = (int)(chain % q.blocks) * (32 * V) + lane * V, ch = min(own, q.D - V);
  const bool ok = own < q.D;
  const uint64_t rate = m.rate() ? get_f32<V>(p.rate + ch) : 0;
  bool far = false;
  if (m.rate()) {
    float r0, r1;
    unf2(rate, r0, r1);
    far = __any_sync(0xffffffffu, !(r0 > -0.5f && r0 <= 0.f && r1 > -0.5f && r1 <= 0.f));
  }
  uint64_t carry = p.h0 != nullptr ? get_f32<V>(p.h0 + (long long)b * q.D + ch) : 0;
  const int tile = W * GL, rounds = (q.S + K * tile - 1) / (K * tile);
  int buf = 0;
  if (K > 1) cluster_sync_all();   // all of them run: their shared memory may be written
  for (int it = 0; it < rounds; ++it) {
    const int t0 = (it * K + rank) * tile + warp * GL;   // (below 2^31: S is at most 2^30)
    const int n = min(GL, q.S - t0);                     // tokens of this run; may be none
    uint64_t a[GL], u[GL];
    Pack<T, V> rz[GL];
    auto tokens = [&](auto full, auto far_) {
      Pack<T, V> rx[GL], rf[GL], ri[GL];
      const T *px = p.x + b * q.xb + t0 * q.xt + ch, *pf = p.f + b * q.fb + t0 * q.ft + ch;
      const T *pi = m.i() ? p.i + b * q.ib + t0 * q.it + ch : nullptr, *pz = m.z() ? p.z + b * q.zb + t0 * q.zt + ch : nullptr;
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        if (!decltype(full)::value && j >= n) break;
        rf[j] = load_pack<T, V>(pf + j * q.ft);
        rx[j] = load_pack<T, V>(px + j * q.xt);
        if (m.i()) ri[j] = load_pack<T, V>(pi + j * q.it);
        if (m.z()) rz[j] = load_pack<T, V>(pz + j * q.zt);
      }
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        a[j] = dup2(1.f), u[j] = 0;
        if (!decltype(full)::value && j >= n) continue;
        const Decay d = gated_decay<T, decltype(far_)::value>(m, pair_of<T, V>(rf[j]), rate);
        a[j] = d.a;
        u[j] = pair_of<T, V>(rx[j]);
        if (m.i()) u[j] = mul2(u[j], logistic_pair2<T>(pair_of<T, V>(ri[j])));
        if (m.scale() == GATED_CONVEX) u[j] = mul2(u[j], d.rest);
        if (m.scale() == GATED_VARIANCE) {
          const uint64_t q2 = rest2_pair(d.a, d.rest);
          u[j] = mul2(u[j], mul2(q2, inv_scale_pair(q2)));
        }
      }
    };
    if (n == GL && !far) tokens(std::true_type{}, std::false_type{});
    else if (n == GL) tokens(std::true_type{}, std::true_type{});
    else tokens(std::false_type{}, std::true_type{});
    Run mine = no_tokens();
#pragma unroll
    for (int j = 0; j < GL; ++j) mine = Run{mul2(a[j], mine.A), fma2(a[j], mine.H, u[j])};
    uint64_t h = gated_exchange<false>(sh, mine, carry, buf, K, rank);
    buf ^= 1;
    if (n <= 0) continue;
    if (p.ckpt != nullptr && ok) put_pair<float, V>(p.ckpt + ((long long)b * q.nc + t0 / GL) * q.D + ch, h);
    T* py = p.y + ((long long)b * q.S + t0) * q.D + ch;
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      if (j >= n) break;
      h = fma2(a[j], h, u[j]);
      uint64_t o = h;
      if (m.z()) {
        const uint64_t z = pair_of<T, V>(rz[j]);
        o = mul2(o, mul2(z, logistic_pair2<T>(z)));
      }
      if (ok) put_pair<T, V>(py + (long long)j * q.D, o);
    }
  }
  if (p.h_last != nullptr && rank == 0 && warp == 0 && ok) put_pair<float, V>(p.h_last + (long long)b * q.D + ch, carry);
}

template <typename T, int V, class M> __global__ void __launch_bounds__(32 * GATED_WARPS) gated_bw(GatedPtrs<T> p, GatedDims q, M m) {
  __shared__ GatedShared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  const int K = q.K, rank = K > 1 ? (int)cluster_rank() : 0;
  const long long chain = blockIdx.x / K;
  const int b = (int)(chain / q.blocks), own = (int)(chain % q.blocks) * (32 * V) + lane * V, ch = min(own, q.D - V);
  const bool ok = own < q.D;
  const uint64_t rate = m.rate() ? get_f32<V>(p.rate + ch) : 0;
  uint64_t carry = p.dh_last != nullptr ? get_f32<V>(p.dh_last + (long long)b * q.D + ch) : 0, drate = 0;
  const int tile = W * GL, rounds = (q.S + K * tile - 1) / (K * tile);
  int buf = 0;
  if (K > 1) cluster_sync_all();   // all of them run: their shared memory may be written
  for (int it = rounds - 1; it >= 0; --it) {
    const int t0 = (it * K + rank) * tile + warp * GL;
    const int n = min(GL, q.S - t0);
    // per token: its factor, what comes in from above, and what dx, di, df, drate have per unit of G or a G
    uint64_t a[GL], up[GL], gx_[GL], gi_[GL], gf_[GL], gr_[GL];
    auto tokens = [&](auto full) {
      Pack<T, V> rx[GL], rf[GL], ri[GL], rz[GL], rg[GL];
      const T *px = p.x + b * q.xb + t0 * q.xt + ch, *pf = p.f + b * q.fb + t0 * q.ft + ch, *pg = p.dy + b * q.gb + t0 * q.gt + ch;
      const T *pi = m.i() ? p.i + b * q.ib + t0 * q.it + ch : nullptr, *pz = m.z() ? p.z + b * q.zb + t0 * q.zt + ch : nullptr;
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        if (!decltype(full)::value && j >= n) break;
        rf[j] = load_pack<T, V>(pf + j * q.ft);
        rx[j] = load_pack<T, V>(px + j * q.xt);
        if (m.i()) ri[j] = load_pack<T, V>(pi + j * q.it);
        if (m.z()) rz[j] = load_pack<T, V>(pz + j * q.zt);
        rg[j] = load_pack<T, V>(pg + j * q.gt);
      }
      uint64_t h = n > 0 ? get_f32<V>(p.ckpt_in + ((long long)b * q.nc + t0 / GL) * q.D + ch) : 0;
#pragma unroll
      for (int j = 0; j < GL; ++j) {
        a[j] = dup2(1.f), up[j] = 0;
        if (!decltype(full)::value && j >= n) continue;
        const Decay d = gated_decay<T, true>(m, pair_of<T, V>(rf[j]), rate);
        a[j] = d.a;
        uint64_t gx = pair_of<T, V>(rx[j]), s = dup2(1.f), cg = 0;
        if (m.i()) {
          uint64_t g;
          logistic_both<T>(pair_of<T, V>(ri[j]), g, cg);
          gx = mul2(g, gx);
          s = g;
        }
        uint64_t w = h, u = gx;
        if (m.scale() == GATED_CONVEX) {
          w = add2(h, neg2(gx));
          u = mul2(gx, d.rest);
          s = mul2(s, d.rest);
        }
        if (m.scale() == GATED_VARIANCE) {
          const uint64_t q2 = rest2_pair(d.a, d.rest), inv = inv_scale_pair(q2), sc = mul2(q2, inv);
          w = add2(h, neg2(mul2(mul2(d.a, gx), inv)));
          u = mul2(gx, sc);
          s = mul2(s, sc);
        }
        gx_[j] = s;
        if (m.i()) gi_[j] = mul2(u, cg);
        if (m.rate()) {
          gr_[j] = mul2(w, d.sf);
          gf_[j] = mul2(mul2(gr_[j], rate), d.cf);
        } else {
          gf_[j] = mul2(w, d.rest);
        }
        h = fma2(d.a, h, u);
        up[j] = pair_of<T, V>(rg[j]);
        if (m.z()) {
          const uint64_t z = pair_of<T, V>(rz[j]);
          uint64_t sz, cz;
          logistic_both<T>(z, sz, cz);
          const uint64_t dz = mul2(mul2(up[j], h), mul2(sz, fma2(z, cz, dup2(1.f))));
          if (ok) put_pair<T, V>(p.dz + ((long long)b * q.S + t0 + j) * q.D + ch, dz);
          up[j] = mul2(up[j], mul2(z, sz));
        }
      }
    };
    if (n == GL) tokens(std::true_type{});
    else tokens(std::false_type{});
    Run mine = no_tokens();
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) mine = Run{mul2(a[j], mine.A), mul2(a[j], add2(up[j], mine.H))};
    uint64_t c = gated_exchange<true>(sh, mine, carry, buf, K, rank);
    buf ^= 1;
    if (n <= 0) continue;
    const long long at = ((long long)b * q.S + t0) * q.D + ch;
#pragma unroll
    for (int j = GL - 1; j >= 0; --j) {
      if (j >= n) continue;
      const uint64_t G = add2(up[j], c);
      c = mul2(a[j], G);
      if (m.rate()) drate = fma2(c, gr_[j], drate);
      if (ok) put_pair<T, V>(p.dx + at + (long long)j * q.D, mul2(G, gx_[j]));
      if (ok) put_pair<T, V>(p.df + at + (long long)j * q.D, mul2(c, gf_[j]));
      if (m.i() && ok) put_pair<T, V>(p.di + at + (long long)j * q.D, mul2(G, gi_[j]));
    }
  }
  if (p.dh0 != nullptr && rank == 0 && warp == 0 && ok) put_pair<float, V>(p.dh0 + (long long)b * q.D + ch, carry);
  if (m.rate() && p.rate_parts != nullptr) {   // over the warps' runs, in order
    __syncthreads();
    sh.part[0][warp][lane].A = drate;
    __syncthreads();
    if (warp == 0 && ok) {
      for (int w = 1; w < W; ++w) drate = add2(drate, sh.part[0][w][lane].A);
      put_pair<float, V>(p.rate_parts + ((long long)b * K + rank) * q.D + ch, drate);
    }
  }
}

template <typename T, int V, class M> int gated_launch(bool back, const GatedPtrs<T>& p, const GatedDims& q, M m, cudaStream_t st) {
  void (*const kern)(GatedPtrs<T>, GatedDims, M) = back ? gated_bw<T, V, M> : gated_fw<T, V, M>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)q.B * q.blocks * q.K));
  cfg.blockDim = dim3(32 * q.warps);
  cfg.stream = st;
  cudaLaunchAttribute at[1] = {};
  if (q.K > 1) {
    if (q.K > 8) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = q.K, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  cfg.attrs = at;
  note_launch();
  MLSTM_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p, q, m));
  return MLSTM_OK;
}

template <typename T> int gated_run(bool back, int V, const GatedPtrs<T>& p, const GatedDims& q, cudaStream_t st) {
  const bool rate = p.rate != nullptr, i = p.i != nullptr, z = p.z != nullptr;
  if (V == 1) return gated_launch<T, 1>(back, p, q, GatedAny{rate, i, z, q.scale}, st);
  auto pick = [&](auto r, auto s, auto ii, auto zz) {
    return gated_launch<T, 2>(back, p, q, GatedFixed<decltype(r)::value, decltype(s)::value, decltype(ii)::value, decltype(zz)::value>{}, st);
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

}  // namespace mlstm
