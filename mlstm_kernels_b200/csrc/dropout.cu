// Dropout whose mask is a function of the element's index, and is never stored:
//
//   y = residual + (w_n >= threshold ? scale x : 0),   scale = 1 / (1 - p), threshold = p 2^32 rounded
//
// w_n, the word of element n of x (in its logical order, whatever its strides), is word n mod 4 of Philox4x32 with seven rounds, the
// fewest that its authors found to pass every test of BigCrush (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as
// 1, 2, 3; 2011), under the key `seed`, of the counter (n div 4, offset).  The backward is the same call on dy.
#include "divide.cuh"
#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

struct DropoutDims {
  long long n;                 // elements
  long long n1, n2, D;         // sizes behind the first axis
  long long xs[3], rs[3], ys[3];   // strides in elements of the axes before the last, of x, residual, y
};

struct DropoutKey {
  const long long* device;     // the seed where it lies on the GPU, else null
  unsigned long long seed, offset;
  unsigned threshold;
  bool some;                   // false: everything is dropped (p = 1)
  float scale;
};

struct Words { unsigned w[4]; };
__device__ __forceinline__ void mul_wide(unsigned a, unsigned b, unsigned& hi, unsigned& lo) {
  unsigned long long r;
  asm("mul.wide.u32 %0, %1, %2;" : "=l"(r) : "r"(a), "r"(b));
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(r));
}
__device__ __forceinline__ Words philox7(unsigned n_lo, unsigned n_hi, unsigned long long offset, unsigned k0, unsigned k1) {
  unsigned c0 = n_lo, c1 = n_hi, c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    unsigned h0, l0, h1, l1;
    mul_wide(c0, 0xD2511F53u, h0, l0);
    mul_wide(c2, 0xCD9E8D57u, h1, l1);
    c0 = h1 ^ c1 ^ k0;
    c1 = l1;
    c2 = h0 ^ c3 ^ k1;
    c3 = l0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

__device__ __forceinline__ unsigned long long seed_of(const DropoutKey& key) {
  return key.device != nullptr ? (unsigned long long)*key.device : key.seed;
}
__device__ __forceinline__ float dropped(float v, unsigned word, const DropoutKey& key) { return word >= key.threshold ? v * key.scale : 0.f; }

// V neighbouring elements to an access of 16 bytes (of the wider type), DROP_U accesses to a thread.  FLAT: all tensors lie in the
// order of their elements; else rows of D, a multiple of V, at strides that are multiples of it.
//
// Memory bounds it, once the generator does not: seven rounds for four elements are 14 wide multiplications and as many three-input
// exclusive ors.  Two bytes read and two written an element leave little for them (8 x 4096 x 2048 bf16 45 us, 5.9 TB/s); with a bf16
// residual 61 us (6.6 TB/s), 4 x 8192 x 4096 with an f32 residual 195 (6.9), without one in 16 bits from heads' layout 53 (5.0).
constexpr int DROP_THREADS = 256, DROP_U = 4;
struct DropoutRows {
  Divide chunks, n2, n1;
  unsigned xs[3], rs[3], ys[3];   // strides in chunks: all tensors end below 2^31 of them
};
struct RowsAt {   // where chunk n lies
  unsigned i0, i1, i2, d;
  __device__ __forceinline__ RowsAt(const DropoutRows& rows, unsigned n) {
    const unsigned r = rows.chunks(n), r1 = rows.n2(r);
    d = n - r * rows.chunks.d, i2 = r - r1 * rows.n2.d, i0 = rows.n1(r1), i1 = r1 - i0 * rows.n1.d;
  }
  __device__ __forceinline__ unsigned operator()(const unsigned (&s)[3]) const { return i0 * s[0] + i1 * s[1] + i2 * s[2] + d; }
};
template <typename T, typename O, int V, bool FLAT, bool RES>
__global__ void __launch_bounds__(DROP_THREADS, 4)
    dropout_wide(const T* __restrict__ x, const O* __restrict__ residual, O* __restrict__ y, long long count, DropoutRows rows, DropoutKey key) {
  constexpr int CHUNKS = DROP_U * DROP_THREADS;   // of a CTA: a power of two
  const long long first = (long long)blockIdx.x * CHUNKS, whole = count / V;
  const unsigned long long quads = (unsigned long long)first * (V / 4), seed = seed_of(key);
  auto work = [&](auto all) {
    Pack<T, V> xv[DROP_U];
    Pack<O, V> rv[DROP_U];
    O* to[DROP_U];
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
      const int c = threadIdx.x + u * DROP_THREADS;
      if (!decltype(all)::value && first + c >= whole) break;
      if constexpr (FLAT) {
        xv[u] = load_pack<T, V>(x + first * V + c * V);
        if (RES) rv[u] = load_pack<O, V>(residual + first * V + c * V);
        to[u] = y + first * V + c * V;
      } else {
        const RowsAt at(rows, (unsigned)first + c);
        xv[u] = load_pack<T, V>(x + (long long)at(rows.xs) * V);
        if (RES) rv[u] = load_pack<O, V>(residual + (long long)at(rows.rs) * V);
        to[u] = y + (long long)at(rows.ys) * V;
      }
    }
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
      const int c = threadIdx.x + u * DROP_THREADS;
      if (!decltype(all)::value && first + c >= whole) break;
      Pack<O, V> o;
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        // The CTA's counters begin at a multiple of their number, a power of two: their high half is one for all, and what the rounds
        // make of it and of the offset alone is worked out once.
        const Words w = philox7((unsigned)quads + c * (V / 4) + k / 4, (unsigned)(quads >> 32), key.offset, (unsigned)seed, (unsigned)(seed >> 32));
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          float v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) v[e] = dropped(to_f32(xv[u].e[k + j + e]), w.w[j + e], key) + (RES ? to_f32(rv[u].e[k + j + e]) : 0.f);
          from_f32x2(v[0], v[1], o.e + k + j);
        }
      }
      store_pack(to[u], o);
    }
  };
  if (first + CHUNKS <= whole) {
    work(std::true_type{});
    return;
  }
  work(std::false_type{});
  const long long n = whole * V + threadIdx.x;   // what is left of a chunk
  if (FLAT && n < count && n / V / CHUNKS == blockIdx.x) {
    const Words w = philox7((unsigned)(n / 4), (unsigned)(n / 4 >> 32), key.offset, (unsigned)seed, (unsigned)(seed >> 32));
    y[n] = from_f32<O>(dropped(to_f32(x[n]), w.w[n % 4], key) + (RES ? to_f32(residual[n]) : 0.f));
  }
}

// For any alignment, and for p = 1: a warp hands its words round, so that neighbouring lanes have neighbouring elements.  Single elements
// are bound by instructions: 8 x 4096 x 2048 bf16, one element off the boundary, 93 us (the kernel above 45), with a residual 101 (60), in
// rows 140.  (Four neighbours to a thread 189 and 211; one or four times 128 elements to a warp 95 and 105.)
constexpr int DROP_ANY = 2;   // times 128 elements to a warp
enum class Lie { FLAT, ROWS, FAR };   // as above, the same in 32-bit offsets of elements, in 64-bit ones
template <typename T, typename O, Lie LIE>
__global__ void __launch_bounds__(DROP_THREADS)
    dropout_any(const T* __restrict__ x, const O* __restrict__ residual, O* __restrict__ y, DropoutDims q, DropoutRows rows, DropoutKey key) {
  constexpr int E = 4 * DROP_ANY;
  using Where = std::conditional_t<LIE == Lie::ROWS, unsigned, long long>;
  __shared__ uint4 words[DROP_THREADS];
  const int lane = threadIdx.x & 31;
  const long long first = ((long long)blockIdx.x * DROP_THREADS + threadIdx.x - lane) * E;   // of this warp
  const unsigned long long seed = seed_of(key);
  const unsigned* const mine = reinterpret_cast<const unsigned*>(words + threadIdx.x - lane) + lane;
  auto work = [&](auto all) {
    float v[E], add[E];
    Where to[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const long long n = first + 32 * j + lane;
      if (!decltype(all)::value && n >= q.n) break;
      Where xa = (Where)n, ra = xa;
      to[j] = xa;
      if constexpr (LIE == Lie::ROWS) {
        const RowsAt at(rows, (unsigned)n);
        xa = at(rows.xs), ra = at(rows.rs), to[j] = at(rows.ys);
      }
      if constexpr (LIE == Lie::FAR) {
        const long long r = n / q.D, d = n - r * q.D, r1 = r / q.n2, i2 = r - r1 * q.n2, i0 = r1 / q.n1, i1 = r1 - i0 * q.n1;
        auto at = [&](const long long (&s)[3]) { return i0 * s[0] + i1 * s[1] + i2 * s[2] + d; };
        xa = at(q.xs), ra = at(q.rs), to[j] = at(q.ys);
      }
      v[j] = to_f32(x[xa]);
      add[j] = residual != nullptr ? to_f32(residual[ra]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < DROP_ANY; ++u) {
      const long long quad = first / 4 + 32 * u + lane;
      const Words w = philox7((unsigned)quad, (unsigned)(quad >> 32), key.offset, (unsigned)seed, (unsigned)(seed >> 32));
      __syncwarp();
      words[threadIdx.x] = make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = 4 * u + k;
        if (!decltype(all)::value && first + 32 * j + lane >= q.n) break;
        y[to[j]] = from_f32<O>((key.some ? dropped(v[j], mine[32 * k], key) : 0.f) + add[j]);
      }
    }
  };
  if (first + 32 * E <= q.n) work(std::true_type{});
  else work(std::false_type{});
}

// Rows in chunks of V elements; false where strides or widths are not multiples of V, or 32-bit offsets do not reach
static bool dropout_rows(const DropoutDims& q, int V, DropoutRows& rows) {
  if (q.D % V != 0 || q.n / V >= (1ll << 31)) return false;
  rows = DropoutRows{divide_by(q.D / V), divide_by(q.n2), divide_by(q.n1), {}, {}, {}};
  const long long n[3] = {q.n / (q.n1 * q.n2 * q.D), q.n1, q.n2};
  struct { const long long* from; unsigned* to; } strides[] = {{q.xs, rows.xs}, {q.rs, rows.rs}, {q.ys, rows.ys}};
  for (const auto& s : strides) {   // (without a residual its strides are zero)
    long long end = q.D / V;
    for (int k = 0; k < 3; ++k) {
      if (s.from[k] < 0 || s.from[k] % V != 0 || s.from[k] / V > (1ll << 31)) return false;
      end += (n[k] - 1) * (s.from[k] / V);
      s.to[k] = (unsigned)(s.from[k] / V);
    }
    if (end >= (1ll << 31)) return false;
  }
  return true;
}

template <typename T, typename O>
static void dropout_run(const T* x, const O* residual, O* y, const DropoutDims& q, const DropoutKey& key, cudaStream_t st) {
  constexpr int V = sizeof(T) == 4 || sizeof(O) == 4 ? 4 : 8;
  const bool flat = q.n == q.D;
  DropoutRows rows{};
  const bool wide = key.some && fits_access(x, sizeof(T) * V) && fits_access(y, sizeof(O) * V) && (residual == nullptr || fits_access(residual, sizeof(O) * V)) &&
                    (flat || dropout_rows(q, V, rows));
  if (!wide) {
    const long long per = 4 * DROP_ANY * DROP_THREADS;
    auto go = [&](auto lie) {
      dropout_any<T, O, decltype(lie)::value><<<(unsigned)((q.n + per - 1) / per), DROP_THREADS, 0, st>>>(x, residual, y, q, rows, key);
    };
    if (flat) go(std::integral_constant<Lie, Lie::FLAT>{});
    else if (dropout_rows(q, 1, rows)) go(std::integral_constant<Lie, Lie::ROWS>{});
    else go(std::integral_constant<Lie, Lie::FAR>{});
    return;
  }
  const long long chunks = (q.n + V - 1) / V, per = DROP_U * DROP_THREADS;
  const unsigned grid = (unsigned)((chunks + per - 1) / per);
  auto go = [&](auto f, auto r) {
    dropout_wide<T, O, V, decltype(f)::value, decltype(r)::value><<<grid, DROP_THREADS, 0, st>>>(x, residual, y, q.n, rows, key);
  };
  if (flat) residual != nullptr ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  else residual != nullptr ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
}

int launch_dropout(const void* x, const long long* xs, const void* residual, const long long* rs, void* y, const long long* ys, const long long* sizes, double p,
                   unsigned long long seed, const long long* seed_device, unsigned long long offset, int dtype, int out_dtype, cudaStream_t st) {
  PhaseScope ps(PH_DROPOUT, st);
  DropoutDims q{sizes[0] * sizes[1] * sizes[2] * sizes[3], sizes[1], sizes[2], sizes[3], {xs[0], xs[1], xs[2]}, {0, 0, 0}, {ys[0], ys[1], ys[2]}};
  if (residual != nullptr)
    for (int k = 0; k < 3; ++k) q.rs[k] = rs[k];
  const double t = nearbyint(p * 4294967296.0);
  const DropoutKey key{seed_device, seed, offset, t < 4294967296.0 ? (unsigned)t : 0u, t < 4294967296.0, t < 4294967296.0 ? (float)(1.0 / (1.0 - p)) : 0.f};
  auto go = [&](auto* t, auto* o) {
    using T = std::remove_pointer_t<decltype(t)>;
    using O = std::remove_pointer_t<decltype(o)>;
    dropout_run<T, O>((const T*)x, (const O*)residual, (O*)y, q, key, st);
  };
  if (out_dtype == MLSTM_F32) {
    MLSTM_DTYPE_SWITCH(dtype, T, go((T*)nullptr, (float*)nullptr);)
  } else if (dtype == MLSTM_F32) {
    MLSTM_DTYPE_SWITCH(out_dtype, O, go((float*)nullptr, (O*)nullptr);)
  } else {
    MLSTM_DTYPE_SWITCH(dtype, T, go((T*)nullptr, (T*)nullptr);)
  }
  MLSTM_LAUNCH_CHECK();
  return MLSTM_OK;
}

}  // namespace mlstm
