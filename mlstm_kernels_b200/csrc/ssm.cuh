// What the forward and the backward of the selective state space scan share: sizes, tiles, and the pass over a tile's operands
// before the recurrence.
#pragma once
#include "launch.cuh"
#include "scan_segments.h"
#include "vec.cuh"

namespace mlstm {

// A CTA has SSM_TT tokens of CH = 256 / LN channels at a time: LN neighbouring lanes share C channels, each lane with four
// states of them.  (Not all states in a thread: more warps for the same sequences, and three shuffles sum four values over the states
// of sixteen.  Eight states: fewer instructions, as many exponentials, and the same time.)
constexpr int SSM_TT = 16;
constexpr int SSM_MAX_N = 128;

struct SsmDims {
  int B, S, D, N, G;
  int Dg, tiles;          // channels of a group; tiles of channels that they take
  int per_cta, parts;     // tiles that a CTA of the backward takes one after the other; CTAs to a group then
  int nseg, seg;          // the sequence in nseg segments of seg tokens (a multiple of SSM_TT), each a CTA of its own
  int rows, row0;         // the backward's launch has `rows` (sequence, segment) at most, from row0 on
  int nt;                 // tiles of SSM_TT tokens in the sequence
  bool softplus;
  bool pairs;             // elements of b and c may be fetched two at a time
  // strides in elements (batch, token; and of b and c the group too) of x, dt, z, b, c, dy; the last axis is contiguous
  long long xb, db, zb, bb, bg, cb, cg, gb;
  int xt, dt, zt, bt, ct, gt;
};

// Where a thread stands: states M sub ... M sub + M - 1 of C channels from `ch` on of the CTA's tile in the recurrence; in the
// passes over whole tiles, V neighbouring channels from `col` of the tokens row, row + ROWS, ...
template <int LN, int V, int C_> struct SsmPlace {
  static constexpr int C = C_, M = 4, H = M / 2, THREADS = 256 / C, WARPS = THREADS / 32;
  static constexpr int CH = 256 / LN, NP = M * LN, LC = 32 / LN;
  static constexpr int PER_ROW = CH / V, ROWS = THREADS / PER_ROW;        // threads to a token; tokens at once
  static constexpr int ITEMS = ROWS >= SSM_TT ? 1 : SSM_TT / ROWS;
  static constexpr int BC = (SSM_TT * NP / 2 + THREADS - 1) / THREADS;   // pairs of b's (and of c's) elements to a thread
  static constexpr int YS = CH + 8 * C;                          // row of a (token, channel) array of sums: the tokens of a warp in different banks
  int sub, chl, ch, warp, tile, g, seg, b, d;
  bool on[C];
  int row, col, dcol;
  bool col_on;
  // nseg: segments that the launch has, from seg0 on; the `turn`-th of per_cta tiles
  __device__ __forceinline__ SsmPlace(const SsmDims& s, int nseg, int seg0, int per_cta = 1, int turn = 0) {
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    sub = lane % LN; chl = lane / LN; ch = C * (warp * LC + chl);
    unsigned k = blockIdx.x;
    const int ctas = per_cta == 1 ? s.tiles : s.parts;
    tile = k % ctas * per_cta + turn; k /= ctas;
    g = k % s.G; k /= s.G;
    k += s.row0;
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

// Where a thread's first element of an operand lies, and the bytes from token to token: an address is one multiplication.
struct SsmSource {
  const char* base;
  int stride;
  template <typename T> __device__ __forceinline__ const T* at(int t) const { return reinterpret_cast<const T*>(base + (long long)t * stride); }
};
template <typename T> __device__ __forceinline__ SsmSource ssm_source(const void* p, long long offset, int tstride) {
  return SsmSource{reinterpret_cast<const char*>(static_cast<const T*>(p) + offset), tstride * (int)sizeof(T)};
}

// The operands of STAGES tiles on their way from memory: ARRS arrays of (token, channel), BCS of (token, state).  Each thread
// copies just what it reads itself, so that its own wait is all that it takes.
template <typename T, typename P, int V, int ARRS, int BCS> struct SsmRing {
  static constexpr int RAW = SSM_TT * P::CH, BCN = SSM_TT * P::NP, STAGE = ARRS * RAW + BCS * BCN;
  // two where a token's channels are 256 bytes or more; the backward's tiles (four arrays) take long enough for two.  (How many CTAs an
  // SM then holds is scan_resident()'s to say: the registers are those of as many, and the number of segments goes by it.)
  static constexpr int STAGES = ARRS == 4 || sizeof(T) * P::CH >= 256 ? 2 : 4;
  static constexpr size_t BYTES = sizeof(T) * STAGE * STAGES;
  T* base;
  __device__ __forceinline__ T* at(int tile) const { return base + (unsigned)tile % STAGES * STAGE; }
  // Zeros where a thread never copies: channels and states past the end, and an array that is not given
  __device__ __forceinline__ void clear(const SsmDims& s, const P& p) const {
#pragma unroll 1
    for (int k = 0; k < STAGES; ++k) {
      T* stage = base + k * STAGE;
      if (!p.col_on && p.row < SSM_TT) {
#pragma unroll
        for (int i = 0; i < ARRS; ++i)
#pragma unroll
          for (int j = 0; j < P::ITEMS; ++j) store_pack<T, V>(stage + i * RAW + (p.row + j * P::ROWS) * P::CH + p.col, zero_pack<T, V>());
      }
#pragma unroll
      for (int i = 0; i < BCS; ++i)
#pragma unroll
        for (int j = 0; j < P::BC; ++j) {
          const int e = 2 * (threadIdx.x + j * P::THREADS), n = e % P::NP;
          T* at = stage + ARRS * RAW + i * BCN + e;
          if (e < BCN && n >= s.N) at[0] = from_f32<T>(0.f);
          if (e < BCN && n + 1 >= s.N) at[1] = from_f32<T>(0.f);
        }
    }
  }
  // array `i` of the tile of tokens t0 ...
  __device__ __forceinline__ void copy(const SsmDims& s, const P& p, int t0, int i, const SsmSource& from) const {
    if (!p.col_on) return;
    T* dst = at(t0 / SSM_TT) + i * RAW + p.row * P::CH + p.col;
    if (t0 + SSM_TT <= s.S) {
#pragma unroll
      for (int j = 0; j < P::ITEMS; ++j) copy_async<T, V>(dst + j * P::ROWS * P::CH, from.at<T>(t0 + p.row + j * P::ROWS), true);
    } else {
#pragma unroll
      for (int j = 0; j < P::ITEMS; ++j) {
        const int t = t0 + p.row + j * P::ROWS;
        copy_async<T, V>(dst + j * P::ROWS * P::CH, from.at<T>(t < s.S ? t : 0), t < s.S);
      }
    }
  }
  // the source of b or c for copy_bc
  static __device__ __forceinline__ SsmSource source_bc(const void* from, const P& p, long long bstride, int tstride, long long gstride) {
    return ssm_source<T>(from, p.b * bstride + p.g * gstride + 2 * threadIdx.x % P::NP, tstride);
  }
  __device__ __forceinline__ void copy_bc(const SsmDims& s, const P& p, int t0, int i, const SsmSource& from) const {
    T* dst = at(t0 / SSM_TT) + ARRS * RAW + i * BCN;
    static_assert(2 * P::THREADS % P::NP == 0, "a thread has the same states in each of its tokens");
    const int n = 2 * threadIdx.x % P::NP;
#pragma unroll
    for (int j = 0; j < P::BC; ++j) {
      const int k = 2 * (threadIdx.x + j * P::THREADS), t = t0 + k / P::NP;
      if (k >= BCN || n >= s.N) continue;
      const bool in = t < s.S;
      const T* a = from.at<T>(in ? t : 0);
      if (sizeof(T) == 2 && s.pairs) {
        copy_async<T, 2>(dst + k, a, in);   // (an even number of states)
      } else {
        copy_async<T, 1>(dst + k, a, in);
        if (n + 1 < s.N) copy_async<T, 1>(dst + k + 1, a + 1, in);
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

// The step of V channels; zero (nothing moves) where `out` is true
template <typename T, int V> __device__ __forceinline__ void ssm_step_v(const float (&dt)[V], const float (&bias)[V], bool softplus, bool out, float (&o)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = dt[i] + bias[i];
  if (softplus) {
    float raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = o[i];
    softplus_v<T, V>(raw, o);
  }
  if (out) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
  }
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

// M values of a row of N at `n`, where n may reach past its end
template <int M> __device__ __forceinline__ void ssm_load(const float* row, int N, int n, float (&o)[M]) {
#pragma unroll
  for (int i = 0; i < M; ++i) o[i] = n + i < N ? row[n + i] : 0.f;
}
// A thread's states of a (channel, state) array, N to a channel, as pairs; zeros where there are none
template <typename P> __device__ __forceinline__ void ssm_load_states(const float* from, const SsmDims& s, const P& p, size_t channel, uint64_t (&o)[P::C][P::H]) {
#pragma unroll
  for (int c = 0; c < P::C; ++c) {
    float v[P::M];
#pragma unroll
    for (int i = 0; i < P::M; ++i) v[i] = 0.f;
    if (from != nullptr && p.on[c]) ssm_load<P::M>(from + (channel + c) * s.N, s.N, P::M * p.sub, v);
#pragma unroll
    for (int i = 0; i < P::H; ++i) o[c][i] = f2(v[2 * i], v[2 * i + 1]);
  }
}
template <typename P> __device__ __forceinline__ void ssm_store_states(float* to, const SsmDims& s, const P& p, size_t channel, const uint64_t (&v)[P::C][P::H]) {
#pragma unroll
  for (int c = 0; c < P::C; ++c) {
    if (!p.on[c]) continue;
    float* row = to + (channel + c) * s.N;
#pragma unroll
    for (int i = 0; i < P::H; ++i) {
      const int n = P::M * p.sub + 2 * i;
      float a, b;
      unf2(v[c][i], a, b);
      if (n < s.N) row[n] = a;
      if (n + 1 < s.N) row[n + 1] = b;
    }
  }
}
// The same in an array of this library, NP to a channel
template <typename P> __device__ __forceinline__ void ssm_get_states(const float* from, const P& p, size_t channel, uint64_t (&o)[P::C][P::H]) {
#pragma unroll
  for (int c = 0; c < P::C; ++c) {
    Pack<uint64_t, P::H> l = {};
    if (p.on[c]) l = load_pack<uint64_t, P::H>(reinterpret_cast<const uint64_t*>(from + (channel + c) * P::NP + P::M * p.sub));
#pragma unroll
    for (int i = 0; i < P::H; ++i) o[c][i] = l.e[i];
  }
}
template <typename P> __device__ __forceinline__ void ssm_put_states(float* to, const P& p, size_t channel, const uint64_t (&v)[P::C][P::H]) {
#pragma unroll
  for (int c = 0; c < P::C; ++c) {
    Pack<uint64_t, P::H> o;
#pragma unroll
    for (int i = 0; i < P::H; ++i) o.e[i] = v[c][i];
    if (p.on[c]) store_pack<uint64_t, P::H>(reinterpret_cast<uint64_t*>(to + (channel + c) * P::NP + P::M * p.sub), o);
  }
}
// b or c of one token, a thread's states as pairs
template <typename P> __device__ __forceinline__ Pack<uint64_t, P::H> ssm_token(const float* s_bc, int t, const P& p) {
  return load_pack<uint64_t, P::H>(reinterpret_cast<const uint64_t*>(s_bc + t * P::NP + P::M * p.sub));
}
// a in powers of two, within f32: a step of zero (a tile's tokens behind the last one have that) times a rate leaves the state as it was
template <typename P> __device__ __forceinline__ void ssm_rates(const float* a, const SsmDims& s, const P& p, uint64_t (&a2)[P::C][P::H]) {
  constexpr float MOST = 3.402823466e38f;
  ssm_load_states(a, s, p, (size_t)p.d, a2);
#pragma unroll
  for (int c = 0; c < P::C; ++c)
#pragma unroll
    for (int i = 0; i < P::H; ++i) {
      float x, y;
      unf2(mul2(a2[c][i], f2(kLog2e, kLog2e)), x, y);
      a2[c][i] = f2(min_nan(max_nan(x, -MOST), MOST), min_nan(max_nan(y, -MOST), MOST));
    }
}
// From what other segments leave behind, in their order: v = 2^(a sum) v + left.  first ... last - 1, or last - 1 ... first (BACK).
// A segment's decay can be beyond f32 where token by token no product is (a state of zero, or a small one, that grows; a large one
// that shrinks): it is multiplied on as four equal factors, none above 2^127, so that zero stays zero and a product is out of range
// only where it is so itself.
template <bool BACK, typename P>
__device__ __forceinline__ void ssm_fold(const float* left, const float* sums, int first, int last, const SsmDims& s, const P& p,
                                         const uint64_t (&a2)[P::C][P::H], uint64_t (&v)[P::C][P::H]) {
#pragma unroll 4
  for (int i = 0; i < last - first; ++i) {
    const int j = BACK ? last - 1 - i : first + i;
    const size_t at = ((size_t)p.b * s.nseg + j) * s.D + p.d;
    uint64_t l[P::C][P::H];
    ssm_get_states(left, p, at, l);
#pragma unroll
    for (int c = 0; c < P::C; ++c) {
      const float sum = p.on[c] ? 0.25f * sums[at + c] : 0.f;
#pragma unroll
      for (int e = 0; e < P::H; ++e) {
        float x, y;
        unf2(mul2(f2(sum, sum), a2[c][e]), x, y);
        const uint64_t q = f2(ex2(min_nan(x, 127.f)), ex2(min_nan(y, 127.f)));
        v[c][e] = fma2(q, mul2(q, mul2(q, mul2(q, v[c][e]))), l[c][e]);
      }
    }
  }
}

// host
template <typename... KArgs, typename... Args>
int ssm_launch(void (*kern)(KArgs...), unsigned threads, size_t smem, bool overlap, unsigned grid, cudaStream_t st, Args... args) {
  if (smem > 48 * 1024) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_pdl(overlap, kern, grid, threads, smem, st, args...);
}
// lanes to a channel, with four states each
inline int ssm_lanes(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32; }
inline int ssm_padded(int N) { return 4 * ssm_lanes(N); }
inline int ssm_tile_channels(int N) { return 256 / ssm_lanes(N); }

ScanSlots ssm_bw_slots(int lanes, int dtype);   // of the backward's kernels

#define SSM_LANES_SWITCH(n, LN, ...)                  \
  switch (n) {                                        \
    case 2: { constexpr int LN = 2; __VA_ARGS__ } break;   \
    case 4: { constexpr int LN = 4; __VA_ARGS__ } break;   \
    case 8: { constexpr int LN = 8; __VA_ARGS__ } break;   \
    case 16: { constexpr int LN = 16; __VA_ARGS__ } break; \
    default: { constexpr int LN = 32; __VA_ARGS__ } break; \
  }

}  // namespace mlstm
