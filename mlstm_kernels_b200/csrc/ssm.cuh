// What the forward and the backward of the selective state space scan share: sizes, tiles, and the pass over a tile's operands
// before the recurrence.
#pragma once
#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

// A CTA has SSM_TT tokens of CH = 256 / LN channels at a time: LN neighbouring lanes share C channels, each lane with four states of
// them.  (Four states a thread, not all of them: as many times the warps for the same sequences, and three shuffles sum four values
// over the states of sixteen.)
constexpr int SSM_TT = 16;
constexpr int SSM_MAX_N = 128;

struct SsmDims {
  int B, S, D, N, G;
  int Dg, tiles;          // channels of a group; CTAs that they take
  int nseg, seg;          // the sequence in nseg segments of seg tokens (a multiple of SSM_TT), each a CTA of its own
  int nt;                 // tiles of SSM_TT tokens in the sequence
  bool softplus;
  bool pairs;             // elements of b and c may be fetched two at a time
  // strides in elements (batch, token; and of b and c the group too); the last axis is contiguous
  long long xb, xt, db, dt, zb, zt, bb, bt, bg, cb, ct, cg, gb, gt;   // x, dt, z, b, c, dy
};

// Where a thread stands: states 4 sub ... 4 sub + 3 of C channels from `ch` on of the CTA's tile in the recurrence; in the
// passes over whole tiles, V neighbouring channels from `col` of the tokens row, row + ROWS, ...
template <int LN, int V, int C_> struct SsmPlace {
  static constexpr int C = C_, THREADS = 256 / C, WARPS = THREADS / 32;
  static constexpr int CH = 256 / LN, NP = 4 * LN, LC = 32 / LN;
  static constexpr int PER_ROW = CH / V, ROWS = THREADS / PER_ROW;        // threads to a token; tokens at once
  static constexpr int ITEMS = ROWS >= SSM_TT ? 1 : SSM_TT / ROWS;
  static constexpr int BC = (SSM_TT * NP / 2 + THREADS - 1) / THREADS;   // pairs of b's (and of c's) elements to a thread
  static constexpr int YS = CH + 8 * C;                          // row of a (token, channel) array of sums: the tokens of a warp in different banks
  int sub, chl, ch, warp, tile, g, seg, b, d;
  bool on[C];
  int row, col, dcol;
  bool col_on;
  // nseg: segments that the launch has, from seg0 on
  __device__ __forceinline__ SsmPlace(const SsmDims& s, int nseg, int seg0) {
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    sub = lane % LN; chl = lane / LN; ch = C * (warp * LC + chl);
    unsigned k = blockIdx.x;
    tile = k % s.tiles; k /= s.tiles;
    g = k % s.G; k /= s.G;
    seg = seg0 + k % nseg;
    b = k / nseg;
#pragma unroll
    for (int c = 0; c < C; ++c) on[c] = tile * CH + ch + c < s.Dg;
    d = g * s.Dg + tile * CH + ch;
    row = threadIdx.x / PER_ROW; col = (threadIdx.x % PER_ROW) * V;
    col_on = tile * CH + col < s.Dg && row < SSM_TT;
    dcol = g * s.Dg + tile * CH + col;
  }
};

// The operands of STAGES tiles on their way from memory: ARRS arrays of (token, channel), BCS of (token, state).  Each thread
// copies just what it reads itself, so that its own wait is all that it takes.
template <typename T, typename P, int V, int ARRS, int BCS> struct SsmRing {
  static constexpr int RAW = SSM_TT * P::CH, BCN = SSM_TT * P::NP, STAGE = ARRS * RAW + BCS * BCN;
  // as many as leave shared memory for the CTAs that registers allow; the backward's tiles (four arrays) take long enough for two
  static constexpr int STAGES = ARRS == 4 || sizeof(T) * P::CH >= 256 ? 2 : 4;
  static constexpr size_t BYTES = sizeof(T) * STAGE * STAGES;
  T* base;
  __device__ __forceinline__ T* at(int tile) const { return base + (unsigned)tile % STAGES * STAGE; }
  // array `i` of the tile of tokens t0 ...: src is the sequence's first element of channel p.dcol
  __device__ __forceinline__ void copy(const SsmDims& s, const P& p, int t0, int i, const void* from, long long bstride, long long tstride) const {
    T* dst = at(t0 / SSM_TT) + i * RAW;
    const T* src = static_cast<const T*>(from) + p.b * bstride;
#pragma unroll
    for (int j = 0; j < P::ITEMS; ++j) {
      const int q = p.row + j * P::ROWS;
      if (q >= SSM_TT) continue;
      const bool ok = p.col_on && t0 + q < s.S;
      copy_async<T, V>(dst + q * P::CH + p.col, ok ? src + (t0 + q) * tstride + p.dcol : src, ok);
    }
  }
  __device__ __forceinline__ void copy_bc(const SsmDims& s, const P& p, int t0, int i, const void* from, long long bstride, long long tstride,
                                          long long gstride) const {
    T* dst = at(t0 / SSM_TT) + ARRS * RAW + i * BCN;
    const T* src = static_cast<const T*>(from) + p.b * bstride + p.g * gstride;
#pragma unroll
    for (int j = 0; j < P::BC; ++j) {
      const int k = 2 * (threadIdx.x + j * P::THREADS), n = k % P::NP, t = t0 + k / P::NP;
      if (k >= BCN) continue;
      const bool in = t < s.S, ok0 = in && n < s.N, ok1 = in && n + 1 < s.N;
      const T* a = ok0 ? src + t * tstride + n : src;
      if (sizeof(T) == 2 && s.pairs) {
        copy_async<T, 2>(dst + k, a, ok0);   // (an even number of states)
      } else {
        copy_async<T, 1>(dst + k, a, ok0);
        copy_async<T, 1>(dst + k + 1, ok1 ? a + 1 : src, ok1);
      }
    }
  }
  // what copy_bc brought, as f32
  __device__ __forceinline__ void put(int tile, int i, float* out) const {
    const T* from = at(tile) + ARRS * RAW + i * BCN;
#pragma unroll
    for (int j = 0; j < P::BC; ++j) {
      const int k = 2 * (threadIdx.x + j * P::THREADS);
      if (k >= BCN) continue;
      float v[2];
      unpack(load_pack<T, 2>(from + k), v);
      *reinterpret_cast<float2*>(out + k) = make_float2(v[0], v[1]);
    }
  }
  // V channels of the thread's j-th token of array i
  __device__ __forceinline__ void get(int tile, int i, int j, const P& p, float (&o)[V]) const {
    unpack(load_pack<T, V>(at(tile) + i * RAW + (p.row + j * P::ROWS) * P::CH + p.col), o);
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

// Sums of four values over the LN lanes that share channels, each step halving the values that a lane still carries: a lane ends
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
template <typename P> __device__ __forceinline__ void ssm_rates(const float* a, const SsmDims& s, const P& p, uint64_t (&a2)[P::C][2]) {
#pragma unroll
  for (int c = 0; c < P::C; ++c) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.on[c]) ssm_load4(a + (size_t)(p.d + c) * s.N, s.N, 4 * p.sub, v);
    a2[c][0] = f2(v[0] * kLog2e, v[1] * kLog2e);
    a2[c][1] = f2(v[2] * kLog2e, v[3] * kLog2e);
  }
}
// From what other segments leave behind, in their order: v = 2^(a sum) v + left.  first ... last - 1, or last - 1 ... first (BACK).
template <bool BACK, typename P>
__device__ __forceinline__ void ssm_fold(const float* left, const float* sums, int first, int last, const SsmDims& s, const P& p,
                                         const uint64_t (&a2)[P::C][2], uint64_t (&v)[P::C][2]) {
#pragma unroll 4
  for (int i = 0; i < last - first; ++i) {
    const int j = BACK ? last - 1 - i : first + i;
#pragma unroll
    for (int c = 0; c < P::C; ++c) {
      if (!p.on[c]) continue;
      const size_t at = ((size_t)p.b * s.nseg + j) * s.D + p.d + c;
      const float sum = sums[at];
      const Pack<uint64_t, 2> l = load_pack<uint64_t, 2>(reinterpret_cast<const uint64_t*>(left + at * P::NP + 4 * p.sub));
      v[c][0] = fma2(ex2_pair(mul2(f2(sum, sum), a2[c][0])), v[c][0], l.e[0]);
      v[c][1] = fma2(ex2_pair(mul2(f2(sum, sum), a2[c][1])), v[c][1], l.e[1]);
    }
  }
}

// host
template <typename... KArgs, typename... Args>
int ssm_launch(void (*kern)(KArgs...), unsigned threads, size_t smem, bool overlap, unsigned grid, cudaStream_t st, Args... args) {
  if (smem > 48 * 1024) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_pdl(overlap, kern, grid, threads, smem, st, args...);
}
// lanes to a channel
inline int ssm_lanes(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32; }

inline int ssm_tile_channels(int N) { return 256 / ssm_lanes(N); }

#define SSM_LANES_SWITCH(n, LN, ...)                  \
  switch (n) {                                        \
    case 2: { constexpr int LN = 2; __VA_ARGS__ } break;   \
    case 4: { constexpr int LN = 4; __VA_ARGS__ } break;   \
    case 8: { constexpr int LN = 8; __VA_ARGS__ } break;   \
    case 16: { constexpr int LN = 16; __VA_ARGS__ } break; \
    default: { constexpr int LN = 32; __VA_ARGS__ } break; \
  }

}  // namespace mlstm
