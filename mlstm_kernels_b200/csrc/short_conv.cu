// Short causal convolution of every channel with its own W taps (2 to 4), optional SiLU, forward, backward, and one token.
//
//   u_t = bias + sum_j w_j x_{t-W+1+j};   y_t = u_t, or u_t sigmoid(u_t)
//   du = dy, or dy sigmoid(u) (1 + u (1 - sigmoid(u)));   dx_t = sum_j w_j du_{t+W-1-j};   dw_j = sum du_t x_{t-W+1+j};   dbias = sum du_t
//
// Tokens before the first are those of x_initial (B, W-1, D), or zeros.  Bound by HBM: x in and y out, in the backward x and dy in
// and dx out.  A thread walks a run of tokens of a few neighbouring channels with the last W tokens in registers; tokens at the
// seam of two runs are read by both (W - 1 of a run's length), mostly from L2.
// bf16, 32768 x 2048, four taps and SiLU: forward 60-62 us (4.4 TB/s; schedulers 57 %, special functions 51 % busy: two of them to an
// element for the logistic function alone), backward with its sums 105 (3.9 TB/s; schedulers 52 %).
#include <type_traits>

#include "launch.cuh"
#include "vec.cuh"

namespace mlstm {

struct ConvDims {
  int B, S, D;
  int runs, run;            // runs of `run` tokens
  long long sb, st;         // strides of x in elements; the channel is the last axis
  long long yb, yt;         // of dy
  int w_dtype;
  bool silu;
};

// V channels as f32: one, or pairs for the packed instructions
template <int V> struct Chan {
  using E = uint64_t;
  static constexpr int N = V / 2;
  E v[N];
};
template <> struct Chan<1> {
  using E = float;
  static constexpr int N = 1;
  E v[1];
};
__device__ __forceinline__ float fma_c(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ uint64_t fma_c(uint64_t a, uint64_t b, uint64_t c) { return fma2(a, b, c); }
__device__ __forceinline__ float mul_c(float a, float b) { return a * b; }
__device__ __forceinline__ uint64_t mul_c(uint64_t a, uint64_t b) { return mul2(a, b); }
__device__ __forceinline__ float add_c(float a, float b) { return a + b; }
__device__ __forceinline__ uint64_t add_c(uint64_t a, uint64_t b) { return add2(a, b); }
__device__ __forceinline__ void all_c(float& r, float x) { r = x; }
__device__ __forceinline__ void all_c(uint64_t& r, float x) { r = f2(x, x); }
template <typename T> __device__ __forceinline__ float logistic_c(float a) { return logistic_f<T>(a); }
template <typename T> __device__ __forceinline__ uint64_t logistic_c(uint64_t a) {
  float x, y;
  unf2(a, x, y);
  return logistic_pair<T>(x, y);
}
template <int V> __device__ __forceinline__ void to_chan(const float (&f)[V], Chan<V>& o) {
  if constexpr (V == 1) {
    o.v[0] = f[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) o.v[i] = f2(f[2 * i], f[2 * i + 1]);
  }
}
template <int V> __device__ __forceinline__ void from_chan(const Chan<V>& c, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = c.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) unf2(c.v[i], f[2 * i], f[2 * i + 1]);
  }
}
template <typename T, int V> __device__ __forceinline__ Chan<V> widen(const Pack<T, V>& p) {
  float f[V];
  unpack(p, f);
  Chan<V> o;
  to_chan<V>(f, o);
  return o;
}
template <typename T, int V> __device__ __forceinline__ Pack<T, V> narrow(const Chan<V>& c) {
  float f[V];
  from_chan<V>(c, f);
  return pack<T, V>(f);
}

// Token t of the padded sequence: x for t >= 0, x_initial (row t + W - 1) or zeros before.
template <typename T, int V, int W>
__device__ __forceinline__ Pack<T, V> conv_token(const T* xb, const T* x0b, long long st, int t, int D) {
  if (t >= 0) return load_pack<T, V>(xb + t * st);
  return x0b != nullptr ? load_pack<T, V>(x0b + (size_t)(t + W - 1) * D) : zero_pack<T, V>();
}

// The taps and the bias of V channels; V > 1 reads the taps, V W neighbours, V at a time.
template <int V, int W> __device__ __forceinline__ void conv_params(const void* w, const void* bias, int dtype, int c, Chan<V> (&wr)[W], Chan<V>& br) {
  float f[W][V], all[W * V], b[V];
  if constexpr (V == 1) {
#pragma unroll
    for (int j = 0; j < W; ++j) all[j] = load_any(w, (size_t)c * W + j, dtype);
    b[0] = bias != nullptr ? load_any(bias, c, dtype) : 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float four[V];
      load_any<V>(w, (size_t)c * W + j * V, dtype, four);
#pragma unroll
      for (int i = 0; i < V; ++i) all[j * V + i] = four[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = 0.f;
    if (bias != nullptr) load_any<V>(bias, c, dtype, b);
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) f[j][i] = all[i * W + j];
#pragma unroll
  for (int j = 0; j < W; ++j) to_chan<V>(f[j], wr[j]);
  to_chan<V>(b, br);
}

// u of one token from the W - 1 tokens before and itself
template <int V, int W>
__device__ __forceinline__ Chan<V> conv_sum(const Chan<V> (&wr)[W], const Chan<V>& br, const Chan<V> (&win)[W - 1], const Chan<V>& x) {
  Chan<V> a;
#pragma unroll
  for (int i = 0; i < Chan<V>::N; ++i) {
    a.v[i] = br.v[i];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) a.v[i] = fma_c(wr[j].v[i], win[j].v[i], a.v[i]);
    a.v[i] = fma_c(wr[W - 1].v[i], x.v[i], a.v[i]);
  }
  return a;
}
template <int V, int W> __device__ __forceinline__ void conv_shift(Chan<V> (&win)[W], const Chan<V>& x) {
#pragma unroll
  for (int j = 0; j + 1 < W; ++j) win[j] = win[j + 1];
  win[W - 1] = x;
}

constexpr int CONV_U = 4;   // tokens at a time

// One thread: V channels of one run of one sequence, threads of neighbouring channels next to each other; CONV_U tokens are on their
// way in registers while as many are worked on.  (Copies to shared memory as in the backward cost more instructions than the wait
// that they save: 32768 x 2048 channels in runs of 48, 71 us against 65.)
template <typename T, int V, int W>
__global__ void __launch_bounds__(256, 3)
conv_fw_kernel(const T* x, const T* x0, const void* w, const void* bias, T* y, T* x_last, ConvDims d) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned nvec = (unsigned)(d.D / V);
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (size_t)nvec * d.runs * d.B) return;
  const unsigned rest = (unsigned)(id / nvec);
  const int c = (int)(id - (size_t)rest * nvec) * V;
  const int b = (int)(rest / (unsigned)d.runs), run = (int)(rest - (unsigned)b * (unsigned)d.runs);
  const int t0 = run * d.run, t1 = min(d.S, t0 + d.run);
  const T* xb = x + b * d.sb + c;
  const T* x0b = x0 != nullptr ? x0 + (size_t)b * (W - 1) * d.D + c : nullptr;
  T* yb = y + (size_t)b * d.S * d.D + c;
  Pack<T, V> in[CONV_U], next[CONV_U];
#pragma unroll
  for (int u = 0; u < CONV_U; ++u) in[u] = load_pack<T, V>(xb + min(t0 + u, t1 - 1) * d.st);
  Chan<V> wr[W], br, win[W - 1];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) win[j] = widen(conv_token<T, V, W>(xb, x0b, d.st, t0 - (W - 1) + j, d.D));
  conv_params<V, W>(w, bias, d.w_dtype, c, wr, br);
  for (int t = t0; t < t1; t += CONV_U) {
    if (t + CONV_U < t1) {
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) next[u] = load_pack<T, V>(xb + min(t + CONV_U + u, t1 - 1) * d.st);
    }
#pragma unroll
    for (int u = 0; u < CONV_U; ++u) {
      const Chan<V> v = widen(in[u]);
      Chan<V> a = conv_sum<V, W>(wr, br, win, v);
      if (d.silu) {
#pragma unroll
        for (int i = 0; i < Chan<V>::N; ++i) a.v[i] = mul_c(a.v[i], logistic_c<T>(a.v[i]));
      }
      conv_shift<V, W - 1>(win, v);
      if (t + u < t1) store_pack<T, V>(yb + (size_t)(t + u) * d.D, narrow<T, V>(a));
    }
#pragma unroll
    for (int u = 0; u < CONV_U; ++u) in[u] = next[u];
  }
  if (x_last != nullptr && t1 == d.S) {
    T* lb = x_last + (size_t)b * (W - 1) * d.D + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_pack<T, V>(lb + (size_t)j * d.D, conv_token<T, V, W>(xb, x0b, d.st, d.S - (W - 1) + j, d.D));
  }
}

// The backward's tokens come into shared memory by asynchronous copies, CONV_U of x and dy at a time and SLOTS times as many ahead;
// each thread copies just what it reads itself, so that its own wait is all that it takes.  (In registers they did not come early
// enough: 32768 x 2048 channels in runs of 64, 381 us against 135.)
template <typename T, int V> struct ConvRing {
  static constexpr int PIECE = sizeof(T) * V, SLOT = 2 * CONV_U * 256 * PIECE;
  static constexpr int SLOTS = sizeof(T) * V > 8 ? 3 : 4;   // two CTAs to an SM
  static constexpr size_t BYTES = (size_t)SLOT * SLOTS;
  char* base;
  __device__ __forceinline__ T* at(int slot, int arr, int u) const {
    return reinterpret_cast<T*>(base + slot * SLOT + ((arr * CONV_U + u) * 256 + threadIdx.x) * PIECE);
  }
};
// CTA: CX threads of V channels each, the other threads runs of tokens; CTA (tile, p) takes the runs p, p + parts, ... of its
// channels, RY = 256 / CX at a time, so that the sums for dw and dbias stay in registers until the end.
// partial: (parts, W + 1, D), the last row for dbias; null when neither is wanted.
template <typename T, int V, int W>
__global__ void __launch_bounds__(256, 2)
conv_bw_kernel(const T* x, const T* x0, const void* w, const void* bias, const T* dy, const T* dlast, T* dx, T* dx0, float* partial,
               ConvDims d, int cx, int tiles) {
  using R = ConvRing<T, V>;
  using C = Chan<V>;
  extern __shared__ __align__(16) char sm[];
  __shared__ float s_sum[256 * V];
  pdl_launch_dependents();
  pdl_wait();
  const R ring{sm};
  const int tile = blockIdx.x % tiles, part = blockIdx.x / tiles, parts = gridDim.x / tiles;
  const int lane = threadIdx.x % cx, ry = threadIdx.x / cx, nry = 256 / cx;
  const int c = (tile * cx + lane) * V;
  C wr[W], br, dw[W], db;
  typename C::E zero, one, minus;
  all_c(zero, 0.f); all_c(one, 1.f); all_c(minus, -1.f);
#pragma unroll
  for (int i = 0; i < C::N; ++i) {
    db.v[i] = zero;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j].v[i] = zero;
  }
  if (c < d.D) {
    conv_params<V, W>(w, bias, d.w_dtype, c, wr, br);
    const unsigned items = (unsigned)d.B * (unsigned)d.runs;
    for (unsigned it = (unsigned)part * nry + ry; it < items; it += (unsigned)parts * nry) {
      const int b = (int)(it / (unsigned)d.runs), run = (int)(it - (unsigned)b * (unsigned)d.runs);
      const int t0 = run * d.run, t1 = min(d.S, t0 + d.run);
      const T* xb = x + b * d.sb + c;
      const T* x0b = x0 != nullptr ? x0 + (size_t)b * (W - 1) * d.D + c : nullptr;
      const T* yb = dy + b * d.yb + c;
      const T* lb = dlast != nullptr ? dlast + (size_t)b * (W - 1) * d.D + c : nullptr;
      T* ob = dx + (size_t)b * d.S * d.D + c;
      T* o0b = dx0 != nullptr ? dx0 + (size_t)b * (W - 1) * d.D + c : nullptr;
      // Tokens t0 ... t1 + W - 2: the last W - 1 belong to the next run (or lie behind the sequence, where du = 0), their du is
      // needed for dx here.  Once du of token t is known, dx of token t - W + 1 is; those in front of the run are the run
      // before's, or x_initial's.
      const int te = t1 + W - 1, tr = min(te, d.S);
      auto fetch = [&](int slot, int t) {
        const T *px = xb + t * d.st, *py = yb + t * d.yt;
        if (t + CONV_U <= tr) {
#pragma unroll
          for (int u = 0; u < CONV_U; ++u) {
            copy_async<T, V>(ring.at(slot, 0, u), px + u * d.st, true);
            copy_async<T, V>(ring.at(slot, 1, u), py + u * d.yt, true);
          }
        } else {
#pragma unroll
          for (int u = 0; u < CONV_U; ++u) {
            const bool ok = t + u < tr;
            copy_async<T, V>(ring.at(slot, 0, u), ok ? px + u * d.st : xb, ok);
            copy_async<T, V>(ring.at(slot, 1, u), ok ? py + u * d.yt : yb, ok);
          }
        }
        cp_commit();
      };
#pragma unroll
      for (int i = 0; i < R::SLOTS; ++i) fetch(i, t0 + i * CONV_U);
      C win[W - 1], du[W];   // the W - 1 inputs before token t; du of tokens t - W + 1 ... t
#pragma unroll
      for (int j = 0; j < W; ++j)
#pragma unroll
        for (int i = 0; i < C::N; ++i) du[j].v[i] = zero;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) win[j] = widen(conv_token<T, V, W>(xb, x0b, d.st, t0 - (W - 1) + j, d.D));
      int slot = 0;
      static_assert(CONV_U >= W - 1, "from the second CONV_U tokens of a run on, every output is one of the run");
      // CONV_U tokens from tb on; INNER: all of them and their outputs are this run's, and none is one of x_last
      auto some = [&](int tb, auto inner) {
        constexpr bool INNER = decltype(inner)::value;
        Pack<T, V> px[CONV_U], py[CONV_U];
        cp_wait<R::SLOTS - 1>();
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          px[u] = load_pack<T, V>(ring.at(slot, 0, u));
          py[u] = load_pack<T, V>(ring.at(slot, 1, u));
        }
        fetch(slot, tb + R::SLOTS * CONV_U);
        slot = slot + 1 == R::SLOTS ? 0 : slot + 1;
        T* out = ob + (long long)(tb - (W - 1)) * d.D;
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          const int t = tb + u;
          const C v = widen(px[u]);
          C k = widen(py[u]);
          if (d.silu) {
            const C a = conv_sum<V, W>(wr, br, win, v);
#pragma unroll
            for (int i = 0; i < C::N; ++i) {
              const auto s = logistic_c<T>(a.v[i]);
              k.v[i] = mul_c(k.v[i], mul_c(s, fma_c(a.v[i], fma_c(s, minus, one), one)));
            }
          }
          if (INNER || t < t1) {
#pragma unroll
            for (int i = 0; i < C::N; ++i) {
              db.v[i] = add_c(db.v[i], k.v[i]);
#pragma unroll
              for (int j = 0; j < W - 1; ++j) dw[j].v[i] = fma_c(k.v[i], win[j].v[i], dw[j].v[i]);
              dw[W - 1].v[i] = fma_c(k.v[i], v.v[i], dw[W - 1].v[i]);
            }
          }
          conv_shift<V, W>(du, k);
          conv_shift<V, W - 1>(win, v);
          C o;   // dx of token t - W + 1
#pragma unroll
          for (int i = 0; i < C::N; ++i) {
            o.v[i] = mul_c(wr[0].v[i], du[W - 1].v[i]);
#pragma unroll
            for (int j = 1; j < W; ++j) o.v[i] = fma_c(wr[j].v[i], du[W - 1 - j].v[i], o.v[i]);
          }
          if (INNER) {
            store_pack<T, V>(out + (size_t)u * d.D, narrow<T, V>(o));
            continue;
          }
          const int to = t - (W - 1);
          if (t >= te || (to < t0 && (run != 0 || o0b == nullptr))) continue;
          const int late = to - (d.S - (W - 1));   // row of x_last that this token became
          if (lb != nullptr && late >= 0) {
            const C e = widen(load_pack<T, V>(lb + (size_t)late * d.D));
#pragma unroll
            for (int i = 0; i < C::N; ++i) o.v[i] = add_c(o.v[i], e.v[i]);
          }
          store_pack<T, V>(to >= 0 ? ob + (size_t)to * d.D : o0b + (size_t)(to + W - 1) * d.D, narrow<T, V>(o));
        }
      };
      for (int tb = t0; tb < te; tb += CONV_U) {
        if (tb > t0 && tb + CONV_U <= t1 && tb + CONV_U <= d.S) some(tb, std::true_type());   // (their outputs end W - 1 tokens before)
        else some(tb, std::false_type());
      }
      cp_wait<0>();
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int j = 0; j <= W; ++j) {   // the CTA's runs together, in their order
    float f[V];
    from_chan<V>(j < W ? dw[j < W ? j : 0] : db, f);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) s_sum[(ry * V + i) * cx + lane] = f[i];
    __syncthreads();
    for (int k = threadIdx.x; k < cx * V; k += 256) {
      const int i = k / cx, l = k % cx, col = (tile * cx + l) * V + i;
      float a = 0.f;
      for (int q = 0; q < nry; ++q) a += s_sum[(q * V + i) * cx + l];
      if (col < d.D) partial[((size_t)part * (W + 1) + j) * d.D + col] = a;
    }
  }
}

// dw (D, W) and dbias (D) from the partial sums, always in the same order
__global__ void __launch_bounds__(256)
conv_param_kernel(const float* partial, int parts, int D, int W, void* dw, void* db, int dtype) {
  __shared__ float s_sum[8][33];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int tiles = (D + 31) / 32;
  const int j = blockIdx.x / tiles, col = (blockIdx.x % tiles) * 32 + lane;
  void* out = j < W ? dw : db;
  if (out == nullptr) return;
  float a = 0.f;
  if (col < D)
    for (int p = g; p < parts; p += 8) a += partial[((size_t)p * (W + 1) + j) * D + col];
  s_sum[g][lane] = a;
  __syncthreads();
  if (g != 0 || col >= D) return;
  a = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) a += s_sum[q][lane];
  store_any(out, j < W ? (size_t)col * W + j : (size_t)col, a, dtype);
}

// One token: before (B, W-1, D) are the tokens in front of it, after those in front of the next (may be the same memory: a
// thread reads its channels' rows before it writes them).
template <typename T, int V, int W>
__global__ void __launch_bounds__(128)
conv_step_kernel(const T* x, const T* before, const void* w, const void* bias, T* y, T* after, int B, int D, int w_dtype, bool silu) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned nvec = (unsigned)(D / V);
  const size_t id = (size_t)blockIdx.x * 128 + threadIdx.x;
  if (id >= (size_t)nvec * B) return;
  const int c = (int)(id % nvec) * V;
  const size_t b = id / nvec;
  Pack<T, V> row[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) row[j] = load_pack<T, V>(before + (b * (W - 1) + j) * D + c);
  row[W - 1] = load_pack<T, V>(x + b * D + c);
  Chan<V> wr[W], br, win[W - 1];
  conv_params<V, W>(w, bias, w_dtype, c, wr, br);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) win[j] = widen(row[j]);
  Chan<V> a = conv_sum<V, W>(wr, br, win, widen(row[W - 1]));
  if (silu) {
#pragma unroll
    for (int i = 0; i < Chan<V>::N; ++i) a.v[i] = mul_c(a.v[i], logistic_c<T>(a.v[i]));
  }
  store_pack<T, V>(y + b * D + c, narrow<T, V>(a));
#pragma unroll
  for (int j = 0; j < W - 1; ++j) store_pack<T, V>(after + (b * (W - 1) + j) * D + c, row[j + 1]);
}

// ---- launchers ----------------------------------------------------------------------------------------
constexpr int CONV_V = 4;   // channels to a thread, where alignment allows

// Tokens to a run (a multiple of four): `slots` runs are worked on at once, and the number that ends the last of them soonest is
// taken, each with eight tokens' time to begin and to end (parameters, the tokens read twice).  32768 x 2048 channels backward: 228
// tokens, one run to a slot, 104 us; 64 tokens, 3.6 to a slot, 130.
static int conv_run(int B, int S, long long slots) {
  int best = S;
  long long least = -1;
  for (int rounds = 1; rounds <= 64; ++rounds) {
    long long runs = slots * rounds / B;
    if (runs < 1) runs = 1;
    if (runs > ceil_div(S, 8)) runs = ceil_div(S, 8);
    const int run = ceil_div((int)((S + runs - 1) / runs), 4) * 4;
    const long long items = (long long)B * ceil_div(S, run), cost = (items + slots - 1) / slots * (run + 8);
    if (least < 0 || cost < least) { least = cost; best = run; }
  }
  return best;
}

struct ConvBwGrid { int run, runs, cx, tiles, parts; };
static ConvBwGrid conv_bw_grid(int B, int S, int D) {
  ConvBwGrid g;
  const int nvec = ceil_div(D, D % CONV_V == 0 ? CONV_V : 1);
  g.cx = 32;
  while (g.cx > 1 && g.cx / 2 >= nvec) g.cx /= 2;
  g.tiles = ceil_div(nvec, g.cx);
  long long parts = 2 * sm_count() / g.tiles;   // no more CTAs than run at once: a few over would take as long again
  if (parts < 1) parts = 1;
  const int rows = 256 / g.cx;
  g.run = conv_run(B, S, parts * rows);
  g.runs = ceil_div(S, g.run);
  const long long needed = ((long long)B * g.runs + rows - 1) / rows;
  g.parts = (int)(parts < needed ? parts : needed);
  return g;
}
// (sized for either access width: the grid depends on it)
size_t short_conv_bw_bytes(int B, int S, int D, int W) {
  const ConvBwGrid g = conv_bw_grid(B, S, D);
  return (size_t)g.parts * (W + 1) * D * sizeof(float);
}

static bool conv_sizes_ok(int B, int S, int D, int W) {
  return B > 0 && S > 0 && D > 0 && W >= 2 && W <= 4 && S < (1 << 30) && (long long)B * S < (1ll << 31) && (long long)D * W < (1ll << 31);
}

template <typename T, int V>
static bool conv_vec(int D, const void* w, const void* bias, const void* const* ptrs, int n, const long long* strides, int m) {
  if (D % V != 0 || !fits_access(w, 16) || !fits_access(bias, 16)) return false;
  const size_t bytes = sizeof(T) * V < 16 ? sizeof(T) * V : 16;
  for (int i = 0; i < n; ++i)
    if (!fits_access(ptrs[i], bytes)) return false;
  for (int i = 0; i < m; ++i)
    if (!stride_fits(strides[i], sizeof(T), bytes)) return false;
  return true;
}

#define CONV_TAPS(RUN) \
  switch (W) {         \
    case 2: RUN(2)     \
    case 3: RUN(3)     \
    default: RUN(4)    \
  }

template <typename T, int V>
static int conv_fw_t(const void* x, const void* x0, const void* w, const void* bias, void* y, void* x_last, int W, const ConvDims& d, cudaStream_t st) {
  const size_t threads = (size_t)(d.D / V) * d.runs * d.B, grid = (threads + 255) / 256;
  if (grid >= (1ull << 31)) return MLSTM_ERR_SHAPE;
#define RUN(TAPS) return launch_pdl(grid <= pdl_max_ctas(), conv_fw_kernel<T, V, TAPS>, (unsigned)grid, 256, 0, st, (const T*)x, (const T*)x0, w, bias, (T*)y, (T*)x_last, d);
  CONV_TAPS(RUN)
#undef RUN
}

int launch_short_conv_fw(const void* x, const long long* xs, const void* x0, const void* w, const void* bias, void* y, void* x_last, int B, int S,
                         int D, int W, bool silu, int dtype, int w_dtype, cudaStream_t st) {
  if (!conv_sizes_ok(B, S, D, W)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_CONV, st);
  const long long room = 768ll * sm_count() / (D % CONV_V == 0 ? D / CONV_V : D);
  const int run = conv_run(B, S, room < 1 ? 1 : room);
  const ConvDims d{B, S, D, ceil_div(S, run), run, xs[0], xs[1], 0, 0, w_dtype, silu};
  const void* ptrs[] = {x, x0, y, x_last};
  MLSTM_DTYPE_SWITCH(dtype, T,
    if (conv_vec<T, CONV_V>(D, w, bias, ptrs, 4, xs, 2)) return conv_fw_t<T, CONV_V>(x, x0, w, bias, y, x_last, W, d, st);
    return conv_fw_t<T, 1>(x, x0, w, bias, y, x_last, W, d, st);)
  return MLSTM_ERR_DTYPE;
}

template <typename... KArgs, typename... Args>
static int conv_bw_run(void (*kern)(KArgs...), size_t smem, unsigned grid, cudaStream_t st, Args... args) {
  if (smem > 40 * 1024) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_pdl(grid <= pdl_max_ctas(), kern, grid, 256, smem, st, args...);
}

template <typename T, int V>
static int conv_bw_t(const void* x, const void* x0, const void* w, const void* bias, const void* dy, const void* dlast, void* dx, void* dx0,
                     float* partial, int W, const ConvDims& d, const ConvBwGrid& g, cudaStream_t st) {
  const unsigned grid = (unsigned)(g.parts * ceil_div(ceil_div(d.D, V), g.cx));
#define RUN(TAPS)                                                                                                                       \
  return conv_bw_run(conv_bw_kernel<T, V, TAPS>, ConvRing<T, V>::BYTES, grid, st, (const T*)x, (const T*)x0, w, bias, (const T*)dy, \
                    (const T*)dlast, (T*)dx, (T*)dx0, partial, d, g.cx, ceil_div(ceil_div(d.D, V), g.cx));
  CONV_TAPS(RUN)
#undef RUN
}

int launch_short_conv_bw(const void* x, const long long* xs, const void* x0, const void* w, const void* bias, const void* dy, const long long* ys,
                         const void* dlast, void* dx, void* dx0, void* dw, void* db, float* partial, int B, int S, int D, int W, bool silu,
                         int dtype, int w_dtype, cudaStream_t st) {
  if (!conv_sizes_ok(B, S, D, W)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_CONV, st);
  const ConvBwGrid g = conv_bw_grid(B, S, D);
  const ConvDims d{B, S, D, g.runs, g.run, xs[0], xs[1], ys[0], ys[1], w_dtype, silu};
  const void* ptrs[] = {x, x0, dy, dlast, dx, dx0};
  const long long strides[] = {xs[0], xs[1], ys[0], ys[1]};
  const bool params = dw != nullptr || db != nullptr;
  float* p = params ? partial : nullptr;
  int rc = MLSTM_ERR_DTYPE;
  MLSTM_DTYPE_SWITCH(dtype, T,
    rc = conv_vec<T, CONV_V>(D, w, bias, ptrs, 6, strides, 4) ? conv_bw_t<T, CONV_V>(x, x0, w, bias, dy, dlast, dx, dx0, p, W, d, g, st)
                                                        : conv_bw_t<T, 1>(x, x0, w, bias, dy, dlast, dx, dx0, p, W, d, g, st);)
  if (rc != MLSTM_OK || !params) return rc;
  const unsigned grid = (unsigned)(ceil_div(D, 32) * (W + 1));
  return launch_pdl(grid <= pdl_max_ctas(), conv_param_kernel, grid, 256, 0, st, (const float*)partial, g.parts, D, W, dw, db, w_dtype);
}

template <typename T, int V>
static int conv_step_t(const void* x, const void* before, const void* w, const void* bias, void* y, void* after, int B, int D, int W, bool silu,
                       int w_dtype, cudaStream_t st) {
  const size_t grid = ((size_t)(D / V) * B + 127) / 128;
  if (grid >= (1ull << 31)) return MLSTM_ERR_SHAPE;
#define RUN(TAPS) return launch_pdl(grid <= pdl_max_ctas(), conv_step_kernel<T, V, TAPS>, (unsigned)grid, 128, 0, st, (const T*)x, (const T*)before, w, bias, (T*)y, (T*)after, B, D, w_dtype, silu);
  CONV_TAPS(RUN)
#undef RUN
}

int launch_short_conv_step(const void* x, const void* before, const void* w, const void* bias, void* y, void* after, int B, int D, int W, bool silu,
                           int dtype, int w_dtype, cudaStream_t st) {
  if (!conv_sizes_ok(B, 1, D, W)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_CONV, st);
  const void* ptrs[] = {x, before, y, after};
  MLSTM_DTYPE_SWITCH(dtype, T,
    if (conv_vec<T, CONV_V>(D, w, bias, ptrs, 4, nullptr, 0)) return conv_step_t<T, CONV_V>(x, before, w, bias, y, after, B, D, W, silu, w_dtype, st);
    return conv_step_t<T, 1>(x, before, w, bias, y, after, B, D, W, silu, w_dtype, st);)
  return MLSTM_ERR_DTYPE;
}

}  // namespace mlstm
