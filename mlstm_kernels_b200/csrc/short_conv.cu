// Short causal convolution of every channel with its own W taps (2 to 4), optional SiLU, forward, backward, and one token.
//
//   u_t = bias + sum_j w_j x_{t-W+1+j};   y_t = u_t, or u_t sigmoid(u_t)
//   du = dy, or dy sigmoid(u) (1 + u (1 - sigmoid(u)));   dx_t = sum_j w_j du_{t+W-1-j};   dw_j = sum du_t x_{t-W+1+j};   dbias = sum du_t
//
// Tokens before the first are those of x_initial (B, W-1, D), or zeros.  Bound by HBM: x in and y out, in the backward x and dy in
// and dx out.  A thread walks a run of tokens of a few neighbouring channels with the last W tokens in registers; tokens at the
// seam of two runs are read by both (W - 1 of a run's length), mostly from L2.
#include "vec.cuh"
#include "launch.cuh"

namespace mlstm {

struct ConvDims {
  int B, S, D;
  int runs, run;            // runs of `run` tokens
  long long sb, st;         // strides of x in elements; the channel is the last axis
  long long yb, yt;         // of dy
  int w_dtype;
  bool silu;
};

// Token t of the padded sequence: x for t >= 0, x_initial (row t + W - 1) or zeros before.
template <typename T, int V, int W>
__device__ __forceinline__ Pack<T, V> conv_token(const T* xb, const T* x0b, long long st, int t, int D) {
  if (t >= 0) return load_pack<T, V>(xb + t * st);
  return x0b != nullptr ? load_pack<T, V>(x0b + (size_t)(t + W - 1) * D) : zero_pack<T, V>();
}

template <int V, int W> __device__ __forceinline__ void conv_params(const void* w, const void* bias, int dtype, int c, float (&wr)[W][V], float (&br)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) wr[j][i] = load_any(w, (size_t)(c + i) * W + j, dtype);
    br[i] = bias != nullptr ? load_any(bias, c + i, dtype) : 0.f;
  }
}

// One thread: V channels of one run of one sequence, threads of neighbouring channels next to each other.
template <typename T, int V, int W>
__global__ void __launch_bounds__(256)
conv_fw_kernel(const T* x, const T* x0, const void* w, const void* bias, T* y, T* x_last, ConvDims d) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned nvec = (unsigned)(d.D / V);
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (size_t)nvec * d.runs * d.B) return;
  const int c = (int)(id % nvec) * V;
  const unsigned rest = (unsigned)(id / nvec);
  const int run = (int)(rest % (unsigned)d.runs), b = (int)(rest / (unsigned)d.runs);
  const int t0 = run * d.run, t1 = min(d.S, t0 + d.run);
  const T* xb = x + b * d.sb + c;
  const T* x0b = x0 != nullptr ? x0 + (size_t)b * (W - 1) * d.D + c : nullptr;
  T* yb = y + (size_t)b * d.S * d.D + c;
  float wr[W][V], br[V], win[W - 1][V];
  conv_params<V, W>(w, bias, d.w_dtype, c, wr, br);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) unpack(conv_token<T, V, W>(xb, x0b, d.st, t0 - (W - 1) + j, d.D), win[j]);
  constexpr int U = 4;   // tokens whose loads are in flight together
  for (int t = t0; t < t1; t += U) {
    Pack<T, V> in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) in[u] = load_pack<T, V>(xb + min(t + u, t1 - 1) * d.st);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[V], o[V];
      unpack(in[u], v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a = br[i];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) a = fmaf(wr[j][i], win[j][i], a);
        a = fmaf(wr[W - 1][i], v[i], a);
        o[i] = d.silu ? a * logistic_f(a) : a;
#pragma unroll
        for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
        win[W - 2][i] = v[i];
      }
      if (t + u < t1) store_pack<T, V>(yb + (size_t)(t + u) * d.D, pack<T, V>(o));
    }
  }
  if (x_last != nullptr && t1 == d.S) {
    T* lb = x_last + (size_t)b * (W - 1) * d.D + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_pack<T, V>(lb + (size_t)j * d.D, conv_token<T, V, W>(xb, x0b, d.st, d.S - (W - 1) + j, d.D));
  }
}

// CTA: CX threads of V channels each, the other threads runs of tokens; CTA (tile, p) takes the runs p, p + parts, ... of its
// channels, RY = 256 / CX at a time, so that the sums for dw and dbias stay in registers until the end.
// partial: (parts, W + 1, D), the last row for dbias; null when neither is wanted.
template <typename T, int V, int W>
__global__ void __launch_bounds__(256)
conv_bw_kernel(const T* x, const T* x0, const void* w, const void* bias, const T* dy, const T* dlast, T* dx, T* dx0, float* partial,
               ConvDims d, int cx, int tiles) {
  __shared__ float s_sum[256 * V];
  pdl_launch_dependents();
  pdl_wait();
  const int tile = blockIdx.x % tiles, part = blockIdx.x / tiles, parts = gridDim.x / tiles;
  const int lane = threadIdx.x % cx, ry = threadIdx.x / cx, nry = 256 / cx;
  const int c = (tile * cx + lane) * V;
  const bool on = c < d.D;
  float wr[W][V], br[V], dw[W][V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][i] = 0.f;
  }
  if (on) {
    conv_params<V, W>(w, bias, d.w_dtype, c, wr, br);
    const unsigned items = (unsigned)d.B * (unsigned)d.runs;
    for (unsigned it = (unsigned)part * nry + ry; it < items; it += (unsigned)parts * nry) {
      const int b = (int)(it / (unsigned)d.runs), run = (int)(it % (unsigned)d.runs);
      const int t0 = run * d.run, t1 = min(d.S, t0 + d.run);
      const T* xb = x + b * d.sb + c;
      const T* x0b = x0 != nullptr ? x0 + (size_t)b * (W - 1) * d.D + c : nullptr;
      const T* yb = dy + b * d.yb + c;
      const T* lb = dlast != nullptr ? dlast + (size_t)b * (W - 1) * d.D + c : nullptr;
      T* ob = dx + (size_t)b * d.S * d.D + c;
      T* o0b = dx0 != nullptr ? dx0 + (size_t)b * (W - 1) * d.D + c : nullptr;
      float win[W - 1][V], du[W][V];   // the W - 1 inputs before token t; du of tokens t - W + 1 ... t
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) du[j][i] = 0.f;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) unpack(conv_token<T, V, W>(xb, x0b, d.st, t0 - (W - 1) + j, d.D), win[j]);
      // Tokens t0 ... t1 + W - 2: the last W - 1 belong to the next run (or lie behind the sequence, where du = 0), their du is
      // needed for dx here.  Once du of token t is known, dx of token t - W + 1 is; those in front of the run are the run
      // before's, or x_initial's.
      const int te = t1 + W - 1;
      for (int t = t0; t < te; ++t) {
        float v[V], g[V];
        if (t < d.S) {
          const Pack<T, V> px = load_pack<T, V>(xb + t * d.st), py = load_pack<T, V>(yb + t * d.yt);
          unpack(px, v);
          unpack(py, g);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = g[i] = 0.f;
        }
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float k = g[i];
          if (d.silu) {
            float a = br[i];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) a = fmaf(wr[j][i], win[j][i], a);
            a = fmaf(wr[W - 1][i], v[i], a);
            const float s = logistic_f(a);
            k *= s * fmaf(a, 1.f - s, 1.f);
          }
          if (t < t1) {
            db[i] += k;
#pragma unroll
            for (int j = 0; j < W - 1; ++j) dw[j][i] = fmaf(k, win[j][i], dw[j][i]);
            dw[W - 1][i] = fmaf(k, v[i], dw[W - 1][i]);
          }
#pragma unroll
          for (int j = 0; j < W - 1; ++j) du[j][i] = du[j + 1][i];
          du[W - 1][i] = k;
          float a = 0.f;
#pragma unroll
          for (int j = 0; j < W; ++j) a = fmaf(wr[j][i], du[W - 1 - j][i], a);   // dx of token t - W + 1
          o[i] = a;
#pragma unroll
          for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
          win[W - 2][i] = v[i];
        }
        const int to = t - (W - 1);
        const int late = to - (d.S - (W - 1));   // row of x_last that this token became
        if (lb != nullptr && late >= 0 && (to >= t0 || run == 0)) {
          float e[V];
          unpack(load_pack<T, V>(lb + (size_t)late * d.D), e);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] += e[i];
        }
        if (to >= t0) store_pack<T, V>(ob + (size_t)to * d.D, pack<T, V>(o));
        else if (run == 0 && o0b != nullptr) store_pack<T, V>(o0b + (size_t)(to + W - 1) * d.D, pack<T, V>(o));
      }
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int j = 0; j <= W; ++j) {   // the CTA's runs together, in their order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) s_sum[(ry * V + i) * cx + lane] = j < W ? dw[j < W ? j : 0][i] : db[i];
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
  float wr[W][V], o[V];
  conv_params<V, W>(w, bias, w_dtype, c, wr, o);
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float v[V];
    unpack(row[j], v);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = fmaf(wr[j][i], v[i], o[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = silu ? o[i] * logistic_f(o[i]) : o[i];
  store_pack<T, V>(y + b * D + c, pack<T, V>(o));
#pragma unroll
  for (int j = 0; j < W - 1; ++j) store_pack<T, V>(after + (b * (W - 1) + j) * D + c, row[j + 1]);
}

// ---- launchers ----------------------------------------------------------------------------------------
constexpr int CONV_BW_V = 4;

struct ConvBwGrid { int run, runs, cx, tiles, parts; };
static ConvBwGrid conv_bw_grid(int B, int S, int D) {
  ConvBwGrid g;
  g.run = 32;
  g.runs = ceil_div(S, g.run);
  const int nvec = ceil_div(D, D % CONV_BW_V == 0 ? CONV_BW_V : 1);
  g.cx = 32;
  while (g.cx > 1 && g.cx / 2 >= nvec) g.cx /= 2;
  g.tiles = ceil_div(nvec, g.cx);
  const long long items = (long long)B * g.runs, rounds = (items + 256 / g.cx - 1) / (256 / g.cx);
  long long parts = ceil_div(2 * sm_count(), g.tiles);
  if (parts > rounds) parts = rounds;
  g.parts = (int)(parts < 1 ? 1 : parts);
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

template <typename T, int V> static bool conv_vec(int D, const void* const* ptrs, int n, const long long* strides, int m) {
  if (D % V != 0) return false;
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
  ConvDims d{B, S, D, 0, 16, xs[0], xs[1], 0, 0, w_dtype, silu};
  d.runs = ceil_div(S, d.run);
  const void* ptrs[] = {x, x0, y, x_last};
  MLSTM_DTYPE_SWITCH(dtype, T,
    if (conv_vec<T, 8>(D, ptrs, 4, xs, 2)) return conv_fw_t<T, 8>(x, x0, w, bias, y, x_last, W, d, st);
    return conv_fw_t<T, 1>(x, x0, w, bias, y, x_last, W, d, st);)
  return MLSTM_ERR_DTYPE;
}

template <typename T, int V>
static int conv_bw_t(const void* x, const void* x0, const void* w, const void* bias, const void* dy, const void* dlast, void* dx, void* dx0,
                     float* partial, int W, const ConvDims& d, const ConvBwGrid& g, cudaStream_t st) {
  const unsigned grid = (unsigned)(g.parts * ceil_div(ceil_div(d.D, V), g.cx));
#define RUN(TAPS)                                                                                                                       \
  return launch_pdl(grid <= pdl_max_ctas(), conv_bw_kernel<T, V, TAPS>, grid, 256, 0, st, (const T*)x, (const T*)x0, w, bias, (const T*)dy, \
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
    rc = conv_vec<T, CONV_BW_V>(D, ptrs, 6, strides, 4) ? conv_bw_t<T, CONV_BW_V>(x, x0, w, bias, dy, dlast, dx, dx0, p, W, d, g, st)
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
    if (conv_vec<T, 4>(D, ptrs, 4, nullptr, 0)) return conv_step_t<T, 4>(x, before, w, bias, y, after, B, D, W, silu, w_dtype, st);
    return conv_step_t<T, 1>(x, before, w, bias, y, after, B, D, W, silu, w_dtype, st);)
  return MLSTM_ERR_DTYPE;
}

}  // namespace mlstm
