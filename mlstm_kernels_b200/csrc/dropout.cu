// Dropout whose mask is a function of the element's index, and is never stored:
//
//   y = residual + (w_n >= threshold ? scale x : 0),   scale = 1 / (1 - p), threshold = p 2^32 rounded
//
// w_n, the word of element n of x (in its logical order, whatever its strides), is word n mod 4 of Philox4x32 with seven rounds, the
// fewest that its authors found to pass every test of BigCrush (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as
// 1, 2, 3; 2011), under the key `seed`, of the counter (n div 4, offset).  The backward is the same call on dy.
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
__device__ __forceinline__ Words philox7(unsigned long long n, unsigned long long offset, unsigned k0, unsigned k1) {
  unsigned c0 = (unsigned)n, c1 = (unsigned)(n >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
    c1 = (unsigned)p1;
    c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
    c3 = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

// four elements to a thread, each read where it lies
template <typename T, typename O>
__global__ void dropout_any(const T* x, const O* residual, O* y, DropoutDims q, DropoutKey key) {
  const long long quad = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (quad * 4 >= q.n) return;
  const unsigned long long seed = key.device != nullptr ? (unsigned long long)*key.device : key.seed;
  const Words w = philox7((unsigned long long)quad, key.offset, (unsigned)seed, (unsigned)(seed >> 32));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long n = quad * 4 + j;
    if (n >= q.n) break;
    const long long d = n % q.D, r = n / q.D, i2 = r % q.n2, r1 = r / q.n2, i1 = r1 % q.n1, i0 = r1 / q.n1;
    const float v = to_f32(x[i0 * q.xs[0] + i1 * q.xs[1] + i2 * q.xs[2] + d]);
    float o = w.w[j] >= key.threshold && key.some ? v * key.scale : 0.f;
    if (residual != nullptr) o += to_f32(residual[i0 * q.rs[0] + i1 * q.rs[1] + i2 * q.rs[2] + d]);
    y[i0 * q.ys[0] + i1 * q.ys[1] + i2 * q.ys[2] + d] = from_f32<O>(o);
  }
}

int launch_dropout(const void* x, const long long* xs, const void* residual, const long long* rs, void* y, const long long* ys, const long long* sizes, double p,
                   unsigned long long seed, const long long* seed_device, unsigned long long offset, int dtype, int out_dtype, cudaStream_t st) {
  PhaseScope ps(PH_DROPOUT, st);
  DropoutDims q{sizes[0] * sizes[1] * sizes[2] * sizes[3], sizes[1], sizes[2], sizes[3], {xs[0], xs[1], xs[2]}, {0, 0, 0}, {ys[0], ys[1], ys[2]}};
  if (residual != nullptr)
    for (int k = 0; k < 3; ++k) q.rs[k] = rs[k];
  const double t = nearbyint(p * 4294967296.0);
  const DropoutKey key{seed_device, seed, offset, t < 4294967296.0 ? (unsigned)t : 0u, t < 4294967296.0, t < 4294967296.0 ? (float)(1.0 / (1.0 - p)) : 0.f};
  const long long quads = (q.n + 3) / 4;
  if ((quads + 255) / 256 > 0x7fffffffll) return MLSTM_ERR_SHAPE;
  const unsigned grid = (unsigned)((quads + 255) / 256);
  auto go = [&](auto* t, auto* o) {
    using T = std::remove_pointer_t<decltype(t)>;
    using O = std::remove_pointer_t<decltype(o)>;
    dropout_any<T, O><<<grid, 256, 0, st>>>((const T*)x, (const O*)residual, (O*)y, q, key);
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
