// Layer norm over the last axis, forward and backward.
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   g = dy w:  dx = rstd (g - mean(g) - xhat mean(g xhat));  dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// Bound by HBM: the forward moves x and y, the backward x, dy and dx.  A row stays in the registers of some lanes of a warp (up to
// 512 elements) or of one CTA, 16 elements a thread (eight took 235 us instead of 158 for the backward of 131072 x 1024), so that the variance is taken about the mean without a second read; sums are
// f32, and up to four more rows are on their way meanwhile.  Rows may lie apart in memory (x seen as (B, S, NH, DH) where it lies as
// (B, NH, S, DH)); every CTA stays with one head, whose weight and bias are read once.
// bf16, 4096 x 8 x 16 heads of 256 read in place: forward 93 us (5.8 TB/s), backward 127 (6.3 TB/s; 252 without the copies ahead) and 5
// for the sums over CTAs, alone; 230-239 one after the other in a stream.  fp16, 8077 rows of 4096: 25-26 us (5.0-5.3 TB/s).  Above
// 8192 elements a row takes 1024 threads, whose 64 registers the backward spills (400-530 bytes): 4096 x 16384 bf16 215 us (1.9 TB/s).
#include "vec.cuh"
#include "launch.cuh"
#include "norm_rows.h"

namespace mlstm {

// The rows of one head: row r at (r / n1) s0 + (r % n1) s1 + head s2.
struct LnRows {
  unsigned n1;
  long long s0, s1, s2;
};
// Every step-th of them, without a division for each
struct LnWalk {
  unsigned r, step, i0, i1, d0, d1;
  __device__ __forceinline__ LnWalk(unsigned n1, unsigned first, unsigned step_) : r(first), step(step_) {
    i0 = first / n1; i1 = first - i0 * n1;
    d0 = step / n1; d1 = step - d0 * n1;
  }
  __device__ __forceinline__ void next(unsigned n1) {
    r += step; i0 += d0; i1 += d1;
    if (i1 >= n1) { i1 -= n1; ++i0; }
  }
  __device__ __forceinline__ long long at(const LnRows& k, int head) const { return i0 * k.s0 + i1 * k.s1 + head * k.s2; }
};

struct LnDims {
  unsigned rows;     // of one head
  int NH, D;
  int parts;         // CTAs of one head
  int param_dtype;
};

// Threads to a row, and rows of a CTA at a time
template <int TPR> struct LnGroup {
  static constexpr int THREADS = TPR <= 32 ? 256 : TPR, ROWS = THREADS / TPR;
};
// CTAs to an SM that the registers are kept for; the grid is that many CTAs to an SM at most, as each goes through rows until there
// are no more (a few CTAs over would take as long again).
constexpr int ln_ctas(int threads, bool backward) {
  const int most = backward ? 512 : 768;
  return threads >= most ? 1 : most / threads;
}

// Sums of K values over the TPR threads of a row; every thread gets them.  `turn` alternates the buffers, so that one barrier does.
template <int TPR, int K> __device__ __forceinline__ void row_sums(float (&v)[K], int& turn) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    __shared__ float s_sum[2][K][WARPS];
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < K; ++i) s_sum[turn][i][threadIdx.x >> 5] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      if constexpr (WARPS <= 8) {   // (each thread adds them up: less latency than shuffles)
        v[i] = s_sum[turn][i][0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) v[i] += s_sum[turn][i][w];
      } else {
        v[i] = s_sum[turn][i][threadIdx.x & (WARPS - 1)];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      }
    }
    turn ^= 1;
  }
}
template <int TPR> __device__ __forceinline__ float row_sum(float a, int& turn) {
  float v[1] = {a};
  row_sums<TPR, 1>(v, turn);
  return v[0];
}

// What a thread has of a row: NQ chunks of 16 bytes, E elements each, with aligned rows (VEC) neighbours, else one lane beside the
// other.  ARRS rows at a time (x, or x and dy) come into shared memory by asynchronous copies, SLOTS of them ahead; each thread
// copies just what it reads itself, so that its own wait is all that it takes.
template <typename T, int TPR, bool VEC, int ARRS, int CTAS> struct LnRing {
  static constexpr int THREADS = LnGroup<TPR>::THREADS, E = 16 / sizeof(T), NQ = LN_V / E, H = E / 2;
  static constexpr int SLOT = ARRS * NQ * THREADS * 16 + (ARRS == 2 ? 2 * THREADS * 4 : 0);
  static constexpr int FIT = (216 * 1024 / CTAS - (ARRS == 2 && TPR <= 32 ? 16 * 1024 : 0)) / SLOT, SLOTS = FIT > 4 ? 4 : FIT < 1 ? 1 : FIT;
  static constexpr size_t BYTES = (size_t)SLOT * SLOTS;
  char* base;
  static __device__ __forceinline__ int col(int t, int q, int e) { return VEC ? (q * TPR + t) * E + e : (q * E + e) * TPR + t; }
  __device__ __forceinline__ T* chunk(int slot, int arr, int q) const {
    return reinterpret_cast<T*>(base + slot * SLOT + ((arr * NQ + q) * THREADS + threadIdx.x) * 16);
  }
  __device__ __forceinline__ T* single(int slot, int arr, int q, int e) const {   // a lane's elements apart: each bank once
    return reinterpret_cast<T*>(base + slot * SLOT + (arr * NQ + q) * THREADS * 16) + e * THREADS + threadIdx.x;
  }
  __device__ __forceinline__ float* stat(int slot, int i) const {
    return reinterpret_cast<float*>(base + slot * SLOT + ARRS * NQ * THREADS * 16) + i * THREADS + threadIdx.x;
  }
  // zeros past the row's end, and everywhere where `ok` is false
  __device__ __forceinline__ void copy(int slot, int arr, const T* row, int t, int D, bool ok) const {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      if (VEC) {
        const int c = col(t, q, 0);
        copy_async<T, E>(chunk(slot, arr, q), ok && c < D ? row + c : row, ok && c < D);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = col(t, q, e);
          copy_async<T, 1>(single(slot, arr, q, e), ok && c < D ? row + c : row, ok && c < D);
        }
      }
    }
  }
  __device__ __forceinline__ void get(int slot, int arr, uint64_t (&o)[NQ][H]) const {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      float f[E];
      if (VEC) {
        unpack(load_pack<T, E>(chunk(slot, arr, q)), f);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = to_f32(*single(slot, arr, q, e));
      }
#pragma unroll
      for (int i = 0; i < H; ++i) o[q][i] = f2(f[2 * i], f[2 * i + 1]);
    }
  }
  static __device__ __forceinline__ void store(T* p, int t, int D, const uint64_t (&o)[NQ][H]) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      float f[E];
#pragma unroll
      for (int i = 0; i < H; ++i) unf2(o[q][i], f[2 * i], f[2 * i + 1]);
      if (VEC) {
        const int c = col(t, q, 0);
        if (c < D) store_pack<T, E>(p + c, pack<T, E>(f));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = col(t, q, e);
          if (c < D) p[c] = from_f32<T>(f[e]);
        }
      }
    }
  }
  static __device__ __forceinline__ void param(const void* p, size_t at, int dtype, int t, int D, uint64_t (&o)[NQ][H], float none) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = p == nullptr ? none : 0.f;
      if (p != nullptr && VEC) {
        const int c = col(t, q, 0);
        if (c < D) load_any<E>(p, at + c, dtype, f);
      } else if (p != nullptr) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = col(t, q, e);
          if (c < D) f[e] = load_any(p, at + c, dtype);
        }
      }
#pragma unroll
      for (int i = 0; i < H; ++i) o[q][i] = f2(f[2 * i], f[2 * i + 1]);
    }
  }
};
__device__ __forceinline__ float sum2(uint64_t v) {
  float a, b;
  unf2(v, a, b);
  return a + b;
}

template <typename T, int TPR, bool VEC> using LnFwRing = LnRing<T, TPR, VEC, 1, ln_ctas(LnGroup<TPR>::THREADS, false)>;
template <typename T, int TPR, bool VEC> using LnBwRing = LnRing<T, TPR, VEC, 2, ln_ctas(LnGroup<TPR>::THREADS, true)>;

template <typename T, int TPR, bool VEC>
__global__ void __launch_bounds__(LnGroup<TPR>::THREADS, ln_ctas(LnGroup<TPR>::THREADS, false))
ln_fw_kernel(const T* x, const void* weight, const void* bias, T* y, float* mean, float* rstd, LnRows xr, LnDims d, float eps) {
  using R = LnFwRing<T, TPR, VEC>;
  constexpr int ROWS = LnGroup<TPR>::ROWS, NQ = R::NQ, H = R::H;
  extern __shared__ __align__(16) char sm[];
  pdl_launch_dependents();
  pdl_wait();
  const R ring{sm};
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const int head = blockIdx.x % d.NH, part = blockIdx.x / d.NH;
  const unsigned step = (unsigned)d.parts * ROWS;
  LnWalk at(xr.n1, part * ROWS + g, step);   // the row to fetch next
  auto fetch = [&](int slot) {
    const bool ok = at.r < d.rows;
    ring.copy(slot, 0, ok ? x + at.at(xr, head) : x, t, d.D, ok);
    cp_commit();
    at.next(xr.n1);
  };
#pragma unroll
  for (int i = 0; i < R::SLOTS; ++i) fetch(i);
  uint64_t w[NQ][H], b[NQ][H];
  R::param(weight, (size_t)head * d.D, d.param_dtype, t, d.D, w, 1.f);
  R::param(bias, (size_t)head * d.D, d.param_dtype, t, d.D, b, 0.f);
  const float inv_n = 1.f / (float)d.D;
  int turn = 0, slot = 0;
  for (unsigned r0 = part * ROWS; r0 < d.rows; r0 += step) {
    const unsigned r = r0 + g;
    uint64_t v[NQ][H], s = 0ull;
    cp_wait<R::SLOTS - 1>();
    ring.get(slot, 0, v);
    fetch(slot);
    slot = slot + 1 == R::SLOTS ? 0 : slot + 1;
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int e = 0; e < H; ++e) s = add2(s, v[i][e]);
    const float mu = row_sum<TPR>(sum2(s), turn) * inv_n;
    s = 0ull;
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int e = 0; e < H; ++e) {
        v[i][e] = add2(v[i][e], f2(-mu, -mu));
        if (VEC) {
          if (R::col(t, i, 0) < d.D) s = fma2(v[i][e], v[i][e], s);
        } else {
          float p, q;
          unf2(v[i][e], p, q);
          p = R::col(t, i, 2 * e) < d.D ? p : 0.f;
          q = R::col(t, i, 2 * e + 1) < d.D ? q : 0.f;
          s = fma2(f2(p, q), f2(p, q), s);
        }
      }
    const float rs = rsqrtf(row_sum<TPR>(sum2(s), turn) * inv_n + eps);
    if (r < d.rows) {
      const size_t out = (size_t)r * d.NH + head;
      if (mean != nullptr && t == 0) { mean[out] = mu; rstd[out] = rs; }
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < H; ++e) v[i][e] = fma2(mul2(v[i][e], f2(rs, rs)), w[i][e], b[i][e]);
      R::store(y + out * d.D, t, d.D, v);
    }
  }
  cp_wait<0>();
}

// partial: (parts, 2, NH, D), the sums of this CTA's rows for dw and db; null when neither is wanted
template <typename T, int TPR, bool VEC>
__global__ void __launch_bounds__(LnGroup<TPR>::THREADS, ln_ctas(LnGroup<TPR>::THREADS, true))
ln_bw_kernel(const T* x, const void* weight, const float* mean, const float* rstd, const T* dy, T* dx, float* partial, LnRows xr,
             LnRows yr, LnRows dr, LnDims d) {
  using R = LnBwRing<T, TPR, VEC>;
  constexpr int THREADS = R::THREADS, ROWS = LnGroup<TPR>::ROWS, NQ = R::NQ, H = R::H, E = R::E;
  extern __shared__ __align__(16) char sm[];
  __shared__ float s_part[ROWS > 1 ? ROWS * LN_V * TPR : 1];
  pdl_launch_dependents();
  pdl_wait();
  const R ring{sm};
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const int head = blockIdx.x % d.NH, part = blockIdx.x / d.NH;
  const unsigned step = (unsigned)d.parts * ROWS;
  LnWalk at(xr.n1, part * ROWS + g, step), now = at;   // the row to fetch next, and the one to work on
  auto fetch = [&](int slot) {
    const bool ok = at.r < d.rows;
    const size_t i = ok ? (size_t)at.r * d.NH + head : 0;
    ring.copy(slot, 0, ok ? x + at.at(xr, head) : x, t, d.D, ok);
    ring.copy(slot, 1, ok ? dy + at.at(yr, head) : dy, t, d.D, ok);
    copy_async<float, 1>(ring.stat(slot, 0), mean + i, ok);
    copy_async<float, 1>(ring.stat(slot, 1), rstd + i, ok);
    cp_commit();
    at.next(xr.n1);
  };
#pragma unroll
  for (int i = 0; i < R::SLOTS; ++i) fetch(i);
  uint64_t w[NQ][H], aw[NQ][H], ab[NQ][H];
  R::param(weight, (size_t)head * d.D, d.param_dtype, t, d.D, w, 1.f);
#pragma unroll
  for (int i = 0; i < NQ; ++i)
#pragma unroll
    for (int e = 0; e < H; ++e) aw[i][e] = ab[i][e] = 0ull;
  const float inv_n = 1.f / (float)d.D;
  int turn = 0, slot = 0;
  for (unsigned r0 = part * ROWS; r0 < d.rows; r0 += step) {
    uint64_t v[NQ][H], u[NQ][H], s1 = 0ull, s2 = 0ull;
    cp_wait<R::SLOTS - 1>();
    ring.get(slot, 0, v);
    ring.get(slot, 1, u);
    const float mu = *ring.stat(slot, 0), rs = *ring.stat(slot, 1);
    fetch(slot);
    slot = slot + 1 == R::SLOTS ? 0 : slot + 1;
    const uint64_t scale = f2(rs, rs), shift = f2(-mu, -mu);
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int e = 0; e < H; ++e) {
        v[i][e] = mul2(add2(v[i][e], shift), scale);   // xhat; a column past D has u = 0 and adds nothing
        aw[i][e] = fma2(u[i][e], v[i][e], aw[i][e]);
        ab[i][e] = add2(ab[i][e], u[i][e]);
        u[i][e] = mul2(u[i][e], w[i][e]);
        s1 = add2(s1, u[i][e]);
        s2 = fma2(u[i][e], v[i][e], s2);
      }
    float c[2] = {sum2(s1), sum2(s2)};
    row_sums<TPR, 2>(c, turn);
    const uint64_t c1 = f2(-c[0] * inv_n, -c[0] * inv_n), c2 = f2(-c[1] * inv_n, -c[1] * inv_n);
    if (now.r < d.rows) {
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < H; ++e) v[i][e] = mul2(scale, fma2(v[i][e], c2, add2(u[i][e], c1)));
      R::store(dx + now.at(dr, head), t, d.D, v);
    }
    now.next(xr.n1);
  }
  cp_wait<0>();
  if (partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = partial + (((size_t)part * 2 + which) * d.NH + head) * d.D;
    float f[NQ][E];
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int e = 0; e < H; ++e) unf2(which == 0 ? aw[i][e] : ab[i][e], f[i][2 * e], f[i][2 * e + 1]);
    if (ROWS > 1) {   // the CTA's groups together, in the order of their rows
      if (which == 1) __syncthreads();
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s_part[(g * LN_V + i * E + e) * TPR + t] = f[i][e];
      __syncthreads();
      for (int k = threadIdx.x; k < LN_V * TPR; k += THREADS) {
        float a = 0.f;
#pragma unroll
        for (int q = 0; q < ROWS; ++q) a += s_part[q * LN_V * TPR + k];
        const int ie = k / TPR, c = R::col(k % TPR, ie / E, ie % E);
        if (c < d.D) out[c] = a;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = R::col(t, i, e);
          if (c < d.D) out[c] = f[i][e];
        }
    }
  }
}

// dw and db from the partial sums, always in the same order: a CTA sums 32 columns, each warp every 32nd part
__global__ void __launch_bounds__(1024)
ln_param_kernel(const float* partial, int parts, size_t cols, void* dw, void* db, int param_dtype) {
  __shared__ float s_sum[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const size_t tiles = (cols + 31) / 32;
  const int which = blockIdx.x >= tiles;
  const size_t first = (blockIdx.x - which * tiles) * 32;
  void* out = which ? db : dw;
  if (out == nullptr) return;
  float a = 0.f;
  if (first + lane < cols) {
#pragma unroll 4
    for (int p = g; p < parts; p += 32) a += partial[((size_t)p * 2 + which) * cols + first + lane];
  }
  s_sum[g][lane] = a;
  __syncthreads();
  a = warp_sum(s_sum[lane][g]);   // warp g: column g
  if (lane == 0 && first + g < cols) store_any(out, first + g, a, param_dtype);
}

// ---- launchers ----------------------------------------------------------------------------------------
// CTAs per head: as many as the GPU has room for at once, no more than there are rows for.
static int ln_parts(long long rows, int NH, int D, bool backward) {
  const int tpr = ln_threads(D), threads = tpr <= 32 ? 256 : tpr;
  const long long per_cta = threads / tpr, room = (long long)sm_count() * ln_ctas(threads, backward);
  // (in the backward every CTA writes two rows of partial sums: four rows of input at least)
  const long long most = (rows + per_cta * (backward ? 4 : 1) - 1) / (per_cta * (backward ? 4 : 1));
  long long parts = room / NH;
  if (parts > most) parts = most;
  return (int)(parts < 1 ? 1 : parts);
}

size_t layer_norm_bw_bytes(long long rows, int NH, int D) { return (size_t)ln_parts(rows, NH, D, true) * 2 * NH * D * sizeof(float); }

template <typename T> static bool ln_vec(const void* const* ptrs, int n, const LnRows* rows, int m, int D) {
  if (!ln_whole_chunks(D, sizeof(T))) return false;
  for (int i = 0; i < n; ++i)
    if (!fits_access(ptrs[i], 16)) return false;
  for (int i = 0; i < m; ++i)
    if (!stride_fits(rows[i].s0, sizeof(T), 16) || !stride_fits(rows[i].s1, sizeof(T), 16) || !stride_fits(rows[i].s2, sizeof(T), 16)) return false;
  return true;
}

#define LN_FORMS(RUN)                                                                                                            \
  switch (ln_threads(D)) {                                                                                                       \
    case 4: RUN(4) case 8: RUN(8) case 16: RUN(16) case 32: RUN(32) case 64: RUN(64) case 96: RUN(96) case 128: RUN(128)         \
    case 160: RUN(160) case 192: RUN(192) case 224: RUN(224) case 256: RUN(256) case 512: RUN(512)                               \
  }                                                                                                                              \
  RUN(1024)

template <typename... KArgs, typename... Args>
static int ln_run(void (*kern)(KArgs...), size_t smem, unsigned threads, unsigned grid, cudaStream_t st, Args... args) {
  if (smem > 32 * 1024) MLSTM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_pdl(grid <= pdl_max_ctas(), kern, grid, threads, smem, st, args...);
}

template <typename T>
static int ln_fw_t(const T* x, const LnRows& xr, const void* w, const void* b, T* y, float* mean, float* rstd, const LnDims& d, float eps, cudaStream_t st) {
  const void* ptrs[] = {x, w, b, y};
  const bool vec = ln_vec<T>(ptrs, 4, &xr, 1, d.D);
  const unsigned grid = (unsigned)d.parts * (unsigned)d.NH;
  const int D = d.D;
#define RUN(TPR)                                                                                                                              \
  return vec ? ln_run(ln_fw_kernel<T, TPR, true>, LnFwRing<T, TPR, true>::BYTES, LnGroup<TPR>::THREADS, grid, st, x, w, b, y, mean, rstd, xr, d, eps) \
             : ln_run(ln_fw_kernel<T, TPR, false>, LnFwRing<T, TPR, false>::BYTES, LnGroup<TPR>::THREADS, grid, st, x, w, b, y, mean, rstd, xr, d, eps);
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
  const int D = d.D;
#define RUN(TPR)                                                                                                                              \
  return vec ? ln_run(ln_bw_kernel<T, TPR, true>, LnBwRing<T, TPR, true>::BYTES, LnGroup<TPR>::THREADS, grid, st, x, w, mean, rstd, dy, dx, partial, xr, yr, dr, d) \
             : ln_run(ln_bw_kernel<T, TPR, false>, LnBwRing<T, TPR, false>::BYTES, LnGroup<TPR>::THREADS, grid, st, x, w, mean, rstd, dy, dx, partial, xr, yr, dr, d);
  LN_FORMS(RUN)
#undef RUN
}

static bool ln_sizes_ok(long long n0, long long n1, int NH, int D) {
  return n0 > 0 && n1 > 0 && NH > 0 && D > 0 && D <= LN_MAX_D && n0 < (1ll << 31) && n1 < (1ll << 31) && n0 * n1 < (1ll << 31) &&
         (long long)NH * D < (1ll << 31);
}
static LnRows ln_rows(long long n0, long long n1, const long long* s) {
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
  return launch_pdl(grid <= pdl_max_ctas(), ln_param_kernel, grid, 1024, 0, st, (const float*)partial, d.parts, cols, dw, db, param_dtype);
}

}  // namespace mlstm
