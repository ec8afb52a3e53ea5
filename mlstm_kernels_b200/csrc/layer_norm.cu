// Layer norm over the last axis, forward and backward.
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   g = dy w:  dx = rstd (g - mean(g) - xhat mean(g xhat));  dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// Bound by HBM: the forward moves x and y, the backward x, dy and dx.  A row stays in the registers of one warp (up to 512
// elements) or one CTA, eight neighbouring elements a thread, so that the variance is taken about the mean without a second
// read; sums are f32.  Rows may lie apart in memory (x seen as (B, S, NH, DH) where it lies as (B, NH, S, DH)); every CTA stays
// with one head, whose weight and bias are read once.
#include "vec.cuh"
#include "launch.cuh"

namespace mlstm {

constexpr int LN_V = 8;            // elements a thread reads at once
constexpr int LN_MAX_D = 16384;    // 1024 threads, twice eight elements

// The rows of one head: row r at (r / n1) s0 + (r % n1) s1 + head s2.
struct LnRows {
  unsigned n1;
  long long s0, s1, s2;
  __device__ __forceinline__ long long at(unsigned r, int head) const {
    const unsigned i0 = r / n1;
    return i0 * s0 + (r - i0 * n1) * s1 + head * s2;
  }
};

struct LnDims {
  unsigned rows;     // of one head
  int NH, D;
  int parts;         // CTAs of one head
  int param_dtype;
};

// Sums of two values over the TPR threads of a row; every thread gets both.  `turn` alternates the buffers, so that one barrier does.
template <int TPR> __device__ __forceinline__ float2 row_sum2(float a, float b, int& turn) {
  a = warp_sum(a); b = warp_sum(b);
  if (TPR == 32) return make_float2(a, b);
  __shared__ float2 s_sum[2][TPR / 32];
  if ((threadIdx.x & 31) == 0) s_sum[turn][threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 v = (threadIdx.x & 31) < TPR / 32 ? s_sum[turn][threadIdx.x & 31] : make_float2(0.f, 0.f);
  turn ^= 1;
  return make_float2(warp_sum(v.x), warp_sum(v.y));
}

// Element e of vector v of this thread: eight neighbours with aligned rows (VEC), else one lane beside the other.
template <int TPR, bool VEC> __device__ __forceinline__ int ln_col(int t, int v, int e) {
  return VEC ? (v * TPR + t) * LN_V + e : (v * LN_V + e) * TPR + t;
}
template <typename T, int NV, int TPR, bool VEC>
__device__ __forceinline__ void ln_load(const T* p, int t, int D, float (&o)[NV][LN_V]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (VEC) {
      const int c = ln_col<TPR, VEC>(t, v, 0);
      const Pack<T, LN_V> k = c < D ? load_pack<T, LN_V>(p + c) : zero_pack<T, LN_V>();
#pragma unroll
      for (int e = 0; e < LN_V; ++e) o[v][e] = to_f32(k.e[e]);
    } else {
#pragma unroll
      for (int e = 0; e < LN_V; ++e) {
        const int c = ln_col<TPR, VEC>(t, v, e);
        o[v][e] = c < D ? to_f32(p[c]) : 0.f;
      }
    }
  }
}
template <typename T, int NV, int TPR, bool VEC>
__device__ __forceinline__ void ln_store(T* p, int t, int D, const float (&o)[NV][LN_V]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (VEC) {
      const int c = ln_col<TPR, VEC>(t, v, 0);
      Pack<T, LN_V> k;
#pragma unroll
      for (int e = 0; e < LN_V; ++e) k.e[e] = from_f32<T>(o[v][e]);
      if (c < D) store_pack<T, LN_V>(p + c, k);
    } else {
#pragma unroll
      for (int e = 0; e < LN_V; ++e) {
        const int c = ln_col<TPR, VEC>(t, v, e);
        if (c < D) p[c] = from_f32<T>(o[v][e]);
      }
    }
  }
}
template <int NV, int TPR, bool VEC>
__device__ __forceinline__ void ln_load_param(const void* p, size_t at, int dtype, int t, int D, float (&o)[NV][LN_V], float none) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = ln_col<TPR, VEC>(t, v, 0);
    if (p != nullptr && VEC && c < D) {
      load_any<LN_V>(p, at + c, dtype, o[v]);
      continue;
    }
#pragma unroll
    for (int e = 0; e < LN_V; ++e) {
      const int ce = ln_col<TPR, VEC>(t, v, e);
      o[v][e] = p == nullptr ? none : !VEC && ce < D ? load_any(p, at + ce, dtype) : 0.f;
    }
  }
}

template <typename T, int NV, int TPR, bool VEC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR)
ln_fw_kernel(const T* x, const void* weight, const void* bias, T* y, float* mean, float* rstd, LnRows xr, LnDims d, float eps) {
  constexpr int GROUPS = TPR == 32 ? 8 : 1;
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const int head = blockIdx.x % d.NH, part = blockIdx.x / d.NH;
  float w[NV][LN_V], b[NV][LN_V];
  ln_load_param<NV, TPR, VEC>(weight, (size_t)head * d.D, d.param_dtype, t, d.D, w, 1.f);
  ln_load_param<NV, TPR, VEC>(bias, (size_t)head * d.D, d.param_dtype, t, d.D, b, 0.f);
  const float inv_n = 1.f / (float)d.D;
  int turn = 0;
  const unsigned step = (unsigned)d.parts * GROUPS;
  for (unsigned r = part * GROUPS + g; r < d.rows; r += step) {
    float v[NV][LN_V];
    ln_load<T, NV, TPR, VEC>(x + xr.at(r, head), t, d.D, v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < LN_V; ++e) s += v[i][e];
    const float mu = row_sum2<TPR>(s, 0.f, turn).x * inv_n;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < LN_V; ++e) {
        v[i][e] -= mu;
        if (ln_col<TPR, VEC>(t, i, e) < d.D) s = fmaf(v[i][e], v[i][e], s);
      }
    const float rs = rsqrtf(row_sum2<TPR>(s, 0.f, turn).x * inv_n + eps);
    const size_t row = (size_t)r * d.NH + head;
    if (mean != nullptr && t == 0) { mean[row] = mu; rstd[row] = rs; }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < LN_V; ++e) v[i][e] = fmaf(v[i][e] * rs, w[i][e], b[i][e]);
    ln_store<T, NV, TPR, VEC>(y + row * d.D, t, d.D, v);
  }
}

// partial: (parts, 2, NH, D), the sums of this CTA's rows for dw and db; null when neither is wanted
template <typename T, int NV, int TPR, bool VEC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR)
ln_bw_kernel(const T* x, const void* weight, const float* mean, const float* rstd, const T* dy, T* dx, float* partial, LnRows xr,
             LnRows yr, LnRows dr, LnDims d) {
  constexpr int GROUPS = TPR == 32 ? 8 : 1;
  __shared__ float s_part[GROUPS > 1 ? GROUPS * NV * LN_V * TPR : 1];
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const int head = blockIdx.x % d.NH, part = blockIdx.x / d.NH;
  float w[NV][LN_V], aw[NV][LN_V], ab[NV][LN_V];
  ln_load_param<NV, TPR, VEC>(weight, (size_t)head * d.D, d.param_dtype, t, d.D, w, 1.f);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < LN_V; ++e) aw[i][e] = ab[i][e] = 0.f;
  const float inv_n = 1.f / (float)d.D;
  int turn = 0;
  const unsigned step = (unsigned)d.parts * GROUPS;
  for (unsigned r = part * GROUPS + g; r < d.rows; r += step) {
    float v[NV][LN_V], u[NV][LN_V];
    ln_load<T, NV, TPR, VEC>(x + xr.at(r, head), t, d.D, v);
    ln_load<T, NV, TPR, VEC>(dy + yr.at(r, head), t, d.D, u);
    const size_t row = (size_t)r * d.NH + head;
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < LN_V; ++e) {
        v[i][e] = (v[i][e] - mu) * rs;             // xhat; a column past D has u = 0 and adds nothing
        aw[i][e] = fmaf(u[i][e], v[i][e], aw[i][e]);
        ab[i][e] += u[i][e];
        u[i][e] *= w[i][e];
        s1 += u[i][e];
        s2 = fmaf(u[i][e], v[i][e], s2);
      }
    const float2 c = row_sum2<TPR>(s1, s2, turn);
    const float c1 = c.x * inv_n, c2 = c.y * inv_n;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < LN_V; ++e) v[i][e] = rs * (u[i][e] - c1 - v[i][e] * c2);
    ln_store<T, NV, TPR, VEC>(dx + dr.at(r, head), t, d.D, v);
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = partial + (((size_t)part * 2 + which) * d.NH + head) * d.D;
    if (GROUPS > 1) {   // the CTA's warps together, in the order of their rows
      if (which == 1) __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < LN_V; ++e) s_part[(g * NV * LN_V + i * LN_V + e) * TPR + t] = which == 0 ? aw[i][e] : ab[i][e];
      __syncthreads();
      for (int k = threadIdx.x; k < NV * LN_V * TPR; k += 256) {
        float a = 0.f;
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) a += s_part[q * NV * LN_V * TPR + k];
        const int lane = k % TPR, ie = k / TPR;
        const int col = ln_col<TPR, VEC>(lane, ie / LN_V, ie % LN_V);
        if (col < d.D) out[col] = a;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < LN_V; ++e) {
          const int col = ln_col<TPR, VEC>(t, i, e);
          if (col < d.D) out[col] = which == 0 ? aw[i][e] : ab[i][e];
        }
    }
  }
}

// dw and db from the partial sums, always in the same order
__global__ void __launch_bounds__(256)
ln_param_kernel(const float* partial, int parts, size_t cols, void* dw, void* db, int param_dtype) {
  __shared__ float s_sum[8][33];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const size_t tiles = (cols + 31) / 32;
  const int which = blockIdx.x >= tiles;
  const size_t col = (blockIdx.x - which * tiles) * 32 + lane;
  void* out = which ? db : dw;
  if (out == nullptr) return;
  float a = 0.f;
  if (col < cols)
    for (int p = g; p < parts; p += 8) a += partial[((size_t)p * 2 + which) * cols + col];
  s_sum[g][lane] = a;
  __syncthreads();
  if (g != 0 || col >= cols) return;
  a = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) a += s_sum[q][lane];
  store_any(out, col, a, param_dtype);
}

// ---- launchers ----------------------------------------------------------------------------------------
// CTAs per head: as many as fill the GPU about eight warps deep in registers' room, no more than there are rows for.
static int ln_parts(long long rows, int NH, int D, bool backward) {
  const int tpr = D <= 512 ? 32 : D <= 1024 ? 128 : D <= 4096 ? 256 : D <= 8192 ? 512 : 1024;
  const long long per_cta = tpr == 32 ? 8 : 1;
  const long long ctas = (long long)sm_count() * (backward ? 512 : 1024) / (tpr == 32 ? 256 : tpr);
  const long long most = (rows + per_cta - 1) / per_cta;
  long long parts = (ctas + NH - 1) / NH;
  if (parts > most) parts = most;
  return (int)(parts < 1 ? 1 : parts);
}

size_t layer_norm_bw_bytes(long long rows, int NH, int D) { return (size_t)ln_parts(rows, NH, D, true) * 2 * NH * D * sizeof(float); }

template <typename T> static bool ln_vec(const void* const* ptrs, int n, const LnRows* rows, int m, int D) {
  if (D % LN_V != 0) return false;
  for (int i = 0; i < n; ++i)
    if (!fits_access(ptrs[i], 16)) return false;
  for (int i = 0; i < m; ++i)
    if (!stride_fits(rows[i].s0, sizeof(T), 16) || !stride_fits(rows[i].s1, sizeof(T), 16) || !stride_fits(rows[i].s2, sizeof(T), 16)) return false;
  return true;
}

#define LN_FORMS(RUN)                                                            \
  if (D <= 256) RUN(1, 32)                                                       \
  if (D <= 512) RUN(2, 32)                                                       \
  if (D <= 1024) RUN(1, 128)                                                     \
  if (D <= 2048) RUN(1, 256)                                                     \
  if (D <= 4096) RUN(2, 256)                                                     \
  if (D <= 8192) RUN(2, 512)                                                     \
  RUN(2, 1024)

template <typename T>
static int ln_fw_t(const T* x, const LnRows& xr, const void* w, const void* b, T* y, float* mean, float* rstd, const LnDims& d, float eps, cudaStream_t st) {
  const void* ptrs[] = {x, w, b, y};
  const bool vec = ln_vec<T>(ptrs, 4, &xr, 1, d.D);
  const unsigned grid = (unsigned)d.parts * (unsigned)d.NH;
  const bool overlap = grid <= pdl_max_ctas();
  const int D = d.D;
#define RUN(NV, TPR)                                                                                                                       \
  return launch_pdl(overlap, vec ? ln_fw_kernel<T, NV, TPR, true> : ln_fw_kernel<T, NV, TPR, false>, grid, TPR == 32 ? 256 : TPR, 0, st, x, w, b, \
                    y, mean, rstd, xr, d, eps);
  LN_FORMS(RUN)
#undef RUN
}

template <typename T>
static int ln_bw_t(const T* x, const LnRows& xr, const void* w, const float* mean, const float* rstd, const T* dy, const LnRows& yr, T* dx,
                   const LnRows& dr, float* partial, const LnDims& d, cudaStream_t st) {
  const void* ptrs[] = {x, w, dy, dx};
  const LnRows rows[] = {xr, yr, dr};
  const bool vec = ln_vec<T>(ptrs, 4, rows, 3, d.D);
  const unsigned grid = (unsigned)d.parts * (unsigned)d.NH;
  const bool overlap = grid <= pdl_max_ctas();
  const int D = d.D;
#define RUN(NV, TPR)                                                                                                                       \
  return launch_pdl(overlap, vec ? ln_bw_kernel<T, NV, TPR, true> : ln_bw_kernel<T, NV, TPR, false>, grid, TPR == 32 ? 256 : TPR, 0, st, x, w, \
                    mean, rstd, dy, dx, partial, xr, yr, dr, d);
  LN_FORMS(RUN)
#undef RUN
}

static bool ln_sizes_ok(long long n0, long long n1, int NH, int D) {
  return n0 > 0 && n1 > 0 && NH > 0 && D > 0 && D <= LN_MAX_D && n0 < (1ll << 31) && n1 < (1ll << 31) && n0 * n1 < (1ll << 31) &&
         (long long)NH * D < (1ll << 31);
}
static LnRows ln_rows(long long n0, long long n1, const long long* s) {
  if (s[0] == n1 * s[1]) return LnRows{(unsigned)(n0 * n1), 0, s[1], s[2]};
  return LnRows{(unsigned)n1, s[0], s[1], s[2]};
}

int launch_layer_norm_fw(const void* x, const long long* xs, const void* w, const void* b, void* y, float* mean, float* rstd, long long n0,
                         long long n1, int NH, int D, int dtype, int param_dtype, float eps, cudaStream_t st) {
  if (!ln_sizes_ok(n0, n1, NH, D)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_NORM, st);
  const LnDims d{(unsigned)(n0 * n1), NH, D, ln_parts(n0 * n1, NH, D, false), param_dtype};
  const LnRows xr = ln_rows(n0, n1, xs);
  MLSTM_DTYPE_SWITCH(dtype, T, return ln_fw_t<T>((const T*)x, xr, w, b, (T*)y, mean, rstd, d, eps, st);)
  return MLSTM_ERR_DTYPE;
}

int launch_layer_norm_bw(const void* x, const long long* xs, const void* w, const float* mean, const float* rstd, const void* dy,
                         const long long* ys, void* dx, const long long* ds, void* dw, void* db, float* partial, long long n0, long long n1,
                         int NH, int D, int dtype, int param_dtype, cudaStream_t st) {
  if (!ln_sizes_ok(n0, n1, NH, D)) return MLSTM_ERR_SHAPE;
  PhaseScope ps(PH_NORM, st);
  const LnDims d{(unsigned)(n0 * n1), NH, D, ln_parts(n0 * n1, NH, D, true), param_dtype};
  const LnRows xr = ln_rows(n0, n1, xs), yr = ln_rows(n0, n1, ys), dr = ln_rows(n0, n1, ds);
  const bool params = dw != nullptr || db != nullptr;
  int rc = MLSTM_ERR_DTYPE;
  MLSTM_DTYPE_SWITCH(dtype, T, rc = ln_bw_t<T>((const T*)x, xr, w, mean, rstd, (const T*)dy, yr, (T*)dx, dr, params ? partial : nullptr, d, st);)
  if (rc != MLSTM_OK || !params) return rc;
  const size_t cols = (size_t)NH * D;
  const unsigned grid = (unsigned)((cols + 31) / 32) * 2;
  return launch_pdl(grid <= pdl_max_ctas(), ln_param_kernel, grid, 256, 0, st, (const float*)partial, d.parts, cols, dw, db, param_dtype);
}

}  // namespace mlstm
