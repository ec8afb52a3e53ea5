// What the forward and the backward of the selective state space scan share: sizes, tiles, and the pass over a tile's operands
// before the recurrence.
#pragma once
#include "f32x2.cuh"
#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

// A CTA of 256 threads has SSM_TT tokens of CH = 256 / LN channels at a time: LN neighbouring lanes share a channel, each with four of
// its states.  (Four states a thread, not all of them: four times the warps for the same sequences, and the sums over the states
// cost three shuffles for four tokens.)
constexpr int SSM_TT = 16;
constexpr int SSM_THREADS = 256;
constexpr int SSM_MAX_N = 128;

struct SsmDims {
  int B, S, D, N, G;
  int Dg, tiles;          // channels of a group; CTAs that they take
  int nseg, seg;          // the sequence in nseg segments of seg tokens (a multiple of SSM_TT), each a CTA of its own
  int nt;                 // tiles of SSM_TT tokens in the sequence
  bool softplus;
  // strides in elements (batch, token; and of b and c the group too); the last axis is contiguous
  long long xb, xt, db, dt, zb, zt, bb, bt, bg, cb, ct, cg, gb, gt;   // x, dt, z, b, c, dy
};

// Where a thread stands: states 4 sub ... 4 sub + 3 of channel `ch` of the CTA's tile in the recurrence; in the passes over whole
// tiles, V neighbouring channels from `col` of the tokens row, row + rows, ...
template <int LN, int V> struct SsmPlace {
  static constexpr int CH = SSM_THREADS / LN, NP = 4 * LN, LC = 32 / LN;
  static constexpr int PER_ROW = CH / V, ROWS = SSM_THREADS / PER_ROW;        // threads to a token; tokens at once
  static constexpr int ITEMS = ROWS >= SSM_TT ? 1 : SSM_TT / ROWS;
  static constexpr int BC = (SSM_TT * NP + SSM_THREADS - 1) / SSM_THREADS;    // elements of b (and of c) a thread fetches
  static constexpr int YS = CH + 32 / (LN < 8 ? LN : 8);                      // row of a (token, channel) array of sums: the lanes' tokens in banks of their own
  int sub, chl, ch, warp, tile, g, seg, b, d;
  bool on;
  int row, col, dcol;
  bool col_on;
  __device__ __forceinline__ SsmPlace(const SsmDims& s) {
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    sub = lane % LN; chl = lane / LN; ch = warp * LC + chl;
    unsigned k = blockIdx.x;
    tile = k % s.tiles; k /= s.tiles;
    g = k % s.G; k /= s.G;
    seg = k % s.nseg;
    b = k / s.nseg;
    on = tile * CH + ch < s.Dg;
    d = g * s.Dg + tile * CH + ch;
    row = threadIdx.x / PER_ROW; col = (threadIdx.x % PER_ROW) * V;
    col_on = tile * CH + col < s.Dg && row < SSM_TT;
    dcol = g * s.Dg + tile * CH + col;
  }
};

// The operands of a tile on their way from memory.
template <typename T, int LN, int V, bool BW, bool WITH_C> struct SsmFetch {
  using P = SsmPlace<LN, V>;
  Pack<T, V> x[P::ITEMS], dt[P::ITEMS], z[P::ITEMS], dy[BW ? P::ITEMS : 1];
  T b[P::BC], c[WITH_C ? P::BC : 1];
  __device__ __forceinline__ void load(const SsmIn& in, const void* dyp, const SsmDims& s, const P& p, int t0, bool with_z) {
    const T *xp = static_cast<const T*>(in.x), *tp = static_cast<const T*>(in.dt), *zp = static_cast<const T*>(in.z);
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
      const int t = t0 + p.row + i * P::ROWS;
      const bool ok = p.col_on && t < s.S;
      x[i] = ok ? load_pack<T, V>(xp + p.b * s.xb + t * s.xt + p.dcol) : zero_pack<T, V>();
      dt[i] = ok ? load_pack<T, V>(tp + p.b * s.db + t * s.dt + p.dcol) : zero_pack<T, V>();
      if (with_z && in.z != nullptr) z[i] = ok ? load_pack<T, V>(zp + p.b * s.zb + t * s.zt + p.dcol) : zero_pack<T, V>();
      if (BW) dy[i] = ok ? load_pack<T, V>(static_cast<const T*>(dyp) + p.b * s.gb + t * s.gt + p.dcol) : zero_pack<T, V>();
    }
    const T *bp = static_cast<const T*>(in.b) + p.b * s.bb + p.g * s.bg, *cp = static_cast<const T*>(in.c) + p.b * s.cb + p.g * s.cg;
#pragma unroll
    for (int i = 0; i < P::BC; ++i) {
      const int k = threadIdx.x + i * SSM_THREADS, n = k % P::NP, t = t0 + k / P::NP;
      const bool ok = n < s.N && t < s.S && k < SSM_TT * P::NP;
      b[i] = ok ? bp[t * s.bt + n] : from_f32<T>(0.f);
      if (WITH_C) c[i] = ok ? cp[t * s.ct + n] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void put_bc(float* s_b, float* s_c) const {
#pragma unroll
    for (int i = 0; i < P::BC; ++i) {
      const int k = threadIdx.x + i * SSM_THREADS;
      if (k < SSM_TT * P::NP) {
        s_b[k] = to_f32(b[i]);
        if (WITH_C) s_c[k] = to_f32(c[i]);
      }
    }
  }
};

// Sums over the LN lanes of a channel of TB values each, one per token: the lane ends with the sum of token sub / (LN / TB).
template <int LN, int TB> __device__ __forceinline__ float lane_sums(float (&v)[TB], int sub) {
  constexpr int REP = LN / TB;
#pragma unroll
  for (int half = TB / 2; half >= 1; half >>= 1) {
    const bool up = (sub & (half * REP)) != 0;
#pragma unroll
    for (int t = 0; t < half; ++t) {
      const float mine = up ? v[t + half] : v[t], theirs = up ? v[t] : v[t + half];
      v[t] = mine + __shfl_xor_sync(0xffffffffu, theirs, half * REP);
    }
  }
#pragma unroll
  for (int o = REP / 2; o >= 1; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

template <int LN> __device__ __forceinline__ void ssm_rates(const float* a, const SsmDims& s, int d, int sub, bool on, float (&a2)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] = on && 4 * sub + i < s.N ? a[(size_t)d * s.N + 4 * sub + i] * kLog2e : 0.f;
}

// host: lanes to a channel
inline int ssm_lanes(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32; }

#define SSM_LANES_SWITCH(n, LN, ...)                  \
  switch (n) {                                        \
    case 2: { constexpr int LN = 2; __VA_ARGS__ } break;   \
    case 4: { constexpr int LN = 4; __VA_ARGS__ } break;   \
    case 8: { constexpr int LN = 8; __VA_ARGS__ } break;   \
    case 16: { constexpr int LN = 16; __VA_ARGS__ } break; \
    default: { constexpr int LN = 32; __VA_ARGS__ } break; \
  }

}  // namespace mlstm
