// What the forward and the backward of the selective state space scan share: sizes, tiles, and the pass over a tile's operands
// before the recurrence.
#pragma once
#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

// A CTA of 128 threads has SSM_TT tokens of CH = 256 / LN channels at a time: LN neighbouring lanes share two channels, each lane
// with four states of both.  (Four states a thread, not all of them: as many times the warps for the same sequences, and three
// shuffles sum four values over the states of sixteen.  Two channels: b and c come from shared memory once for both, which a
// wave of 128 bytes a clock bounds.)
constexpr int SSM_TT = 16;
constexpr int SSM_THREADS = 128, SSM_WARPS = SSM_THREADS / 32;
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

// Where a thread stands: states 4 sub ... 4 sub + 3 of the channels `ch` and `ch` + 1 of the CTA's tile in the recurrence; in the
// passes over whole tiles, V neighbouring channels from `col` of the tokens row, row + ROWS, ...
template <int LN, int V> struct SsmPlace {
  static constexpr int CH = 2 * SSM_THREADS / LN, NP = 4 * LN, LC = 32 / LN;
  static constexpr int PER_ROW = CH / V, ROWS = SSM_THREADS / PER_ROW;        // threads to a token; tokens at once
  static constexpr int ITEMS = ROWS >= SSM_TT ? 1 : SSM_TT / ROWS;
  static constexpr int BC = (SSM_TT * NP + SSM_THREADS - 1) / SSM_THREADS;    // elements of b (and of c) a thread fetches
  static constexpr int YS = CH + 16;                             // row of a (token, channel) array of sums: two tokens' in different banks
  int sub, chl, ch, warp, tile, g, seg, b, d;
  bool on[2];
  int row, col, dcol;
  bool col_on;
  // nseg: segments that the launch has, from seg0 on
  __device__ __forceinline__ SsmPlace(const SsmDims& s, int nseg, int seg0) {
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    sub = lane % LN; chl = lane / LN; ch = 2 * (warp * LC + chl);
    unsigned k = blockIdx.x;
    tile = k % s.tiles; k /= s.tiles;
    g = k % s.G; k /= s.G;
    seg = seg0 + k % nseg;
    b = k / nseg;
    on[0] = tile * CH + ch < s.Dg;
    on[1] = tile * CH + ch + 1 < s.Dg;
    d = g * s.Dg + tile * CH + ch;
    row = threadIdx.x / PER_ROW; col = (threadIdx.x % PER_ROW) * V;
    col_on = tile * CH + col < s.Dg && row < SSM_TT;
    dcol = g * s.Dg + tile * CH + col;
  }
};

// b and c of a tile on their way from memory
template <typename T, int LN, int V, bool WITH_C> struct SsmFetchBC {
  using P = SsmPlace<LN, V>;
  T b[P::BC], c[WITH_C ? P::BC : 1];
  __device__ __forceinline__ void load(const SsmIn& in, const SsmDims& s, const P& p, int t0) {
    const T *bp = static_cast<const T*>(in.b) + p.b * s.bb + p.g * s.bg, *cp = static_cast<const T*>(in.c) + p.b * s.cb + p.g * s.cg;
#pragma unroll
    for (int i = 0; i < P::BC; ++i) {
      const int k = threadIdx.x + i * SSM_THREADS, n = k % P::NP, t = t0 + k / P::NP;
      const bool ok = n < s.N && t < s.S && k < SSM_TT * P::NP;
      b[i] = ok ? bp[t * s.bt + n] : from_f32<T>(0.f);
      if (WITH_C) c[i] = ok ? cp[t * s.ct + n] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void put(float* s_b, float* s_c) const {
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

// The step of V channels; zero (nothing moves) where `ok` is false
template <int V> __device__ __forceinline__ void ssm_step_v(const float (&dt)[V], const float (&bias)[V], bool softplus, bool ok, float (&o)[V]) {
  float raw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) raw[i] = dt[i] + bias[i];
  if (softplus) softplus_v<V>(raw, o);
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = !ok ? 0.f : softplus ? o[i] : raw[i];
}

// Sums of four values over the LN lanes of a channel pair, each step halving the values that a lane still carries: a lane ends
// with LEFT of them, from number `first` on.
template <int LN> struct LaneSums {
  static constexpr int LEFT = LN >= 4 ? 1 : 4 / LN;
  static constexpr int SAME = LN >= 4 ? LN / 4 : 1;      // lanes that end with the same value
  static __device__ __forceinline__ int run(float (&v)[4], int sub) {
    int first = 0;
#pragma unroll
    for (int bit = LN / 2, n = 4; bit >= 1; bit >>= 1) {
      if (n > 1) {
        n >>= 1;
        const bool up = (sub & bit) != 0;
#pragma unroll
        for (int j = 0; j < n; ++j) {
          const float mine = up ? v[j + n] : v[j], theirs = up ? v[j] : v[j + n];
          v[j] = mine + __shfl_xor_sync(0xffffffffu, theirs, bit);
        }
        first += up ? n : 0;
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
      }
    }
    return first;
  }
};

// Four values of a row of N at `n`, where n may reach past its end
__device__ __forceinline__ void ssm_load4(const float* row, int N, int n, float (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = n + i < N ? row[n + i] : 0.f;
}
// a in powers of two, as pairs of states
template <int LN, int V> __device__ __forceinline__ void ssm_rates(const float* a, const SsmDims& s, const SsmPlace<LN, V>& p, uint64_t (&a2)[2][2]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.on[c]) ssm_load4(a + (size_t)(p.d + c) * s.N, s.N, 4 * p.sub, v);
    a2[c][0] = f2(v[0] * kLog2e, v[1] * kLog2e);
    a2[c][1] = f2(v[2] * kLog2e, v[3] * kLog2e);
  }
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t v) {
  float a, b;
  unf2(v, a, b);
  return f2(ex2(a), ex2(b));
}
// From what other segments leave behind, in their order: v = 2^(a sum) v + left.  first ... last - 1, or last - 1 ... first (BACK).
template <int LN, int V, bool BACK>
__device__ __forceinline__ void ssm_fold(const float* left, const float* sums, int first, int last, const SsmDims& s, const SsmPlace<LN, V>& p,
                                         const uint64_t (&a2)[2][2], uint64_t (&v)[2][2]) {
#pragma unroll 4
  for (int i = 0; i < last - first; ++i) {
    const int j = BACK ? last - 1 - i : first + i;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (!p.on[c]) continue;
      const size_t at = ((size_t)p.b * s.nseg + j) * s.D + p.d + c;
      const float sum = sums[at];
      const Pack<uint64_t, 2> l = load_pack<uint64_t, 2>(reinterpret_cast<const uint64_t*>(left + at * (4 * LN) + 4 * p.sub));
      v[c][0] = fma2(ex2_pair(mul2(f2(sum, sum), a2[c][0])), v[c][0], l.e[0]);
      v[c][1] = fma2(ex2_pair(mul2(f2(sum, sum), a2[c][1])), v[c][1], l.e[1]);
    }
  }
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
