// Gated linear recurrence: how sequences are divided among CTAs, the calls of the kernels (gated_tiles.cuh), and the step for one
// token.
#include <algorithm>

#include "gated.cuh"

namespace mlstm {

// drate, the sums of n rows of D at `stride` rows, 32 channels and RATE_ROWS rows to a CTA of 32 warps.  Its sum takes the place of its
// first row, for a call on those rows, or, if `out` is given, is the result.  A thread has eight
// loads under way.  (All rows by one CTA: 65536 sequences of 8 tokens of 64 channels take 420 us backward, instead of 184.)
constexpr int RATE_ROWS = 512;
__global__ void __launch_bounds__(1024) gated_rate_sum(float* parts, float* out, int n, int stride, int D, int across) {
  __shared__ float sums[32][33];
  const int part = blockIdx.x / across, c0 = (blockIdx.x - part * across) * 32, rows = min(RATE_ROWS, n - part * RATE_ROWS);
  const long long row = (long long)stride * D;
  float* const first = parts + part * (RATE_ROWS * row);
  float s = 0.f;
  if (c0 + threadIdx.x < D) {
#pragma unroll 8
    for (int k = threadIdx.y; k < rows; k += 32) s += first[c0 + threadIdx.x + k * row];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();   // (all rows of this CTA's channels have been read)
  s = warp_sum(sums[threadIdx.x][threadIdx.y]);   // warp y: channel y's sums
  if (threadIdx.x == 0 && c0 + threadIdx.y < D) (out != nullptr ? out : first)[c0 + threadIdx.y] = s;
}

// The step: V neighbouring channels to a thread, all from one sequence: 4, by accesses of 8 or 16 bytes, where widths and alignments
// allow, else 1.  Bound by memory: 4096 x 4096 (z, "convex", bf16) at 6.1 TB/s, 512 x 4096 6.3 us (with one channel 17); a few
// sequences are one launch.
template <typename T, int V>
__global__ void __launch_bounds__(256) gated_one(const T* x, const T* f, const T* i, const T* z, const float* rate, const float* h, T* y, float* h_new, long long n,
                                                 Divide row, bool small, GatedAny m) {
  const long long k = ((long long)blockIdx.x * 256 + threadIdx.x) * V;
  if (k >= n) return;
  const Pack<T, V> px = load_pack<T, V>(x + k), pf = load_pack<T, V>(f + k);
  const Pack<float, V> ph = load_pack<float, V>(h + k);
  Pack<T, V> pi, pz;
  Pack<float, V> pr;
  if (m.i()) pi = load_pack<T, V>(i + k);
  if (m.z()) pz = load_pack<T, V>(z + k);
  if (m.rate()) {
    const long long first = k / V, d = small ? first - (long long)row((unsigned)first) * row.d : first % row.d;
    pr = load_pack<float, V>(rate + d * V);
  }
  float out[V], state[V];
  auto pair = [](const auto& p, int j) { return f2(to_f32(p.e[j]), to_f32(p.e[V > 1 ? j + 1 : j])); };
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const Run t = gated_token<T, true>(m, pair(pf, j), pair(px, j), m.i() ? pair(pi, j) : 0, m.rate() ? pair(pr, j) : 0);
    const uint64_t v = through(t, pair(ph, j));
    uint64_t o = v;
    if (m.z()) o = mul2(o, mul2(pair(pz, j), logistic_pair2<T>(pair(pz, j))));
    float rest;
    unf2(v, state[j], V > 1 ? state[j + 1] : rest);
    unf2(o, out[j], V > 1 ? out[j + 1] : rest);
  }
  store_pack(h_new + k, pack<float, V>(state));
  store_pack(y + k, pack<T, V>(out));
}

// ---- calls --------------------------------------------------------------------------------------------
// CTAs that run at once, by which groups are cut: those of the 16-bit forward for all.  (The backward and the element-by-element kernels
// hold two to an SM, f32 one to three: their groups are longer than what is under way.)
static int gated_slots() { return 3 * sm_count(); }

bool gated_sizes_ok(int B, int S, int D) {
  return B > 0 && S > 0 && S <= (1 << 30) && D > 0 && D <= (1 << 30) && gated_plan(B, S, D, gated_slots()).units < (1ll << 31);
}
size_t gated_ckpt_bytes(int B, int S, int D) { return (size_t)B * ceil_div(S, GATED_CK) * D * sizeof(float); }
size_t gated_bytes(int B, int S, int D, bool backward) {
  return gated_scratch(gated_plan(B, S, D, gated_slots()), B, D, backward).bytes;
}

int gated_run_f32(bool back, bool rows, const void* ptrs, const GatedDims& q, cudaStream_t st);
int gated_run_bf16(bool back, bool rows, const void* ptrs, const GatedDims& q, cudaStream_t st);
int gated_run_f16(bool back, bool rows, const void* ptrs, const GatedDims& q, cudaStream_t st);
int gated_status_f32(int reset, int* status);
int gated_status_bf16(int reset, int* status);
int gated_status_f16(int reset, int* status);
int gated_status(int reset, int* status) {
  *status = 0;
  for (auto* of : {gated_status_f32, gated_status_bf16, gated_status_f16}) {
    int one = 0;
    const int rc = of(reset, &one);
    if (rc != MLSTM_OK) return rc;
    if (*status == 0) *status = one;
  }
  return MLSTM_OK;
}

struct GatedVoid {   // as GatedPtrs, of any type
  const void *x, *f, *i, *z, *dy;
  const float *rate, *h0, *ckpt_in, *dh_last;
  void *y, *dx, *df, *di, *dz;
  float *h_last, *ckpt, *dh0, *rate_parts;
};
// Rows by 16 bytes where all of them begin on such a boundary, and eight tokens lie within 2^31 bytes
static bool gated_rows(const GatedVoid& p, const long long* st, const long long* gs, int D, int el) {
  const int e = 16 / el;
  if (D % e != 0 || D > (1 << 26)) return false;
  for (const void* a : {p.x, p.f, p.i, p.z, p.dy, (const void*)p.y, (const void*)p.dx, (const void*)p.df, (const void*)p.di, (const void*)p.dz,
                        (const void*)p.rate, (const void*)p.h0, (const void*)p.ckpt_in, (const void*)p.dh_last, (const void*)p.h_last, (const void*)p.ckpt,
                        (const void*)p.dh0, (const void*)p.rate_parts})
    if (!fits_access(a, 16)) return false;
  const void* const ins[4] = {p.x, p.f, p.i, p.z};
  for (int k = 0; k < 8; ++k)
    if (ins[k / 2] != nullptr && (st[k] % e != 0 || st[k] < 0 || (k % 2 == 1 && st[k] > (1 << 26)))) return false;
  return gs == nullptr || (gs[0] % e == 0 && gs[1] % e == 0 && gs[0] >= 0 && gs[1] >= 0 && gs[1] <= (1 << 26));
}
// Looks at memory of a wait: some seconds.  For tests a thread may ask that its next call waits for less, and in vain.
constexpr unsigned GATED_LOOKS = 1u << 24;
struct GatedExpiry { unsigned looks; int units; };
static thread_local GatedExpiry t_expiry{0, 0};
int gated_expiry_selftest(unsigned looks, int units) {
  if (looks > 1000000u || units < 0 || units > 255 || (looks == 0) != (units == 0)) return MLSTM_ERR_UNSUPPORTED;
  t_expiry = GatedExpiry{looks, units};
  return MLSTM_OK;
}

static int gated_call(bool back, GatedVoid p, const long long* st, const long long* gs, void* scratch, int B, int S, int D, int scale, int dtype, float* drate,
                      cudaStream_t stream) {
  PhaseScope ps(PH_GATED, stream);
  const bool rows = gated_rows(p, st, gs, D, (int)dtype_size(dtype));
  const GatedPlan plan = gated_plan(B, S, D, gated_slots());
  const GatedScratch at = gated_scratch(plan, B, D, back);
  unsigned char* const base = static_cast<unsigned char*>(scratch);
  GatedDims q{};
  const GatedExpiry expiry = t_expiry;
  t_expiry = GatedExpiry{0, 0};
  q.looks = expiry.units > 0 ? expiry.looks : GATED_LOOKS;
  q.S = S, q.D = D, q.scale = scale, q.nc = ceil_div(S, GATED_CK);
  q.warps = plan.warps, q.nt = plan.nt, q.group = plan.group, q.groups = plan.groups, q.units = (int)plan.units;
  q.chains = divide_by(plan.chains), q.blocks = divide_by(plan.blocks);
  if (plan.nt > 1) {
    q.ticket = reinterpret_cast<unsigned*>(base);
    q.gave_up = q.ticket + 32;
    q.state = reinterpret_cast<uint2*>(base + at.state);
    q.agg = reinterpret_cast<uint4*>(base + at.agg);
    MLSTM_CUDA_CHECK(cudaMemsetAsync(base, 0, at.rate, stream));
    if (expiry.units > 0) MLSTM_CUDA_CHECK(cudaMemsetAsync(q.ticket, expiry.units, 1, stream));   // (its lowest byte: nobody takes the first units)
  }
  if (drate != nullptr) p.rate_parts = reinterpret_cast<float*>(base + at.rate);
  long long* const to[8] = {&q.xb, &q.xt, &q.fb, &q.ft, &q.ib, &q.it, &q.zb, &q.zt};
  for (int k = 0; k < 8; ++k) *to[k] = st[k];
  if (gs != nullptr) q.gb = gs[0], q.gt = gs[1];
  auto go = [&](auto* t, auto run) {
    using T = std::remove_pointer_t<decltype(t)>;
    const GatedPtrs<T> v{(const T*)p.x, (const T*)p.f, (const T*)p.i, (const T*)p.z, (const T*)p.dy, p.rate, p.h0, p.ckpt_in, p.dh_last, (T*)p.y, (T*)p.dx,
                         (T*)p.df, (T*)p.di, (T*)p.dz, p.h_last, p.ckpt, p.dh0, p.rate_parts};
    return run(back, rows, &v, q, stream);
  };
  int rc = MLSTM_OK;
  if (dtype == MLSTM_F32) rc = go((float*)nullptr, gated_run_f32);
  else if (dtype == MLSTM_BF16) rc = go((__nv_bfloat16*)nullptr, gated_run_bf16);
  else rc = go((__half*)nullptr, gated_run_f16);
  if (rc == MLSTM_OK && drate != nullptr) {
    const int across = ceil_div(D, 32);
    int n = B * q.nt, stride = 1;
    for (int ctas;; n = ctas, stride *= RATE_ROWS) {   // (stride stays below B nt, which is below 2^31)
      ctas = (int)((n + RATE_ROWS - 1ll) / RATE_ROWS);
      gated_rate_sum<<<ctas * across, dim3(32, 32), 0, stream>>>(p.rate_parts, ctas == 1 ? drate : nullptr, n, stride, D, across);
      MLSTM_LAUNCH_CHECK();
      if (ctas == 1) break;
    }
  }
  return rc;
}

int launch_gated_fw(const GatedIn& in, const long long* strides, void* y, float* h_last, float* ckpt, void* scratch, int B, int S, int D, int scale,
                    int dtype, cudaStream_t st) {
  GatedVoid p{in.x, in.f, in.i, in.z, nullptr, in.rate, in.h0, nullptr, nullptr, y, nullptr, nullptr, nullptr, nullptr, h_last, ckpt, nullptr, nullptr};
  return gated_call(false, p, strides, nullptr, scratch, B, S, D, scale, dtype, nullptr, st);
}

int launch_gated_bw(const GatedIn& in, const long long* strides, const float* ckpt, const void* dy, const long long* gs, const float* dh_last, void* dx,
                    void* df, void* di, void* dz, float* drate, float* dh0, void* scratch, int B, int S, int D, int scale, int dtype, cudaStream_t st) {
  GatedVoid p{in.x, in.f, in.i, in.z, dy, in.rate, nullptr, ckpt, dh_last, nullptr, dx, df, di, dz, nullptr, nullptr, dh0, nullptr};
  return gated_call(true, p, strides, gs, scratch, B, S, D, scale, dtype, drate, st);
}

int launch_gated_step(const GatedIn& in, const float* h, void* y, float* h_new, int B, int D, int scale, int dtype, cudaStream_t st) {
  PhaseScope ps(PH_GATED, st);
  const long long n = (long long)B * D;
  const size_t el = dtype_size(dtype);
  bool four = D % 4 == 0;
  for (const void* p : {in.x, in.f, in.i, in.z, (const void*)y}) four = four && fits_access(p, 4 * el);
  for (const float* p : {in.rate, h, (const float*)h_new}) four = four && fits_access(p, 16);
  auto go = [&](auto* t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int V = decltype(v)::value;
    const long long chunks = n / V;
    gated_one<T, V><<<(unsigned)((chunks + 255) / 256), 256, 0, st>>>((const T*)in.x, (const T*)in.f, (const T*)in.i, (const T*)in.z, in.rate, h, (T*)y, h_new, n,
                                                                        divide_by(D / V), chunks < (1ll << 31), GatedAny{in.rate != nullptr, in.i != nullptr, in.z != nullptr, scale});
  };
  MLSTM_DTYPE_SWITCH(dtype, T, if (four) go((T*)nullptr, std::integral_constant<int, 4>{}); else go((T*)nullptr, std::integral_constant<int, 1>{});)
  MLSTM_LAUNCH_CHECK();
  return MLSTM_OK;
}

}  // namespace mlstm
