// Division by a number that is known when a kernel is launched, as in Granlund and Montgomery, Division by invariant integers using
// multiplication (1994).
#pragma once
#include <cuda_runtime.h>

namespace mlstm {

// n / d for n < 2^31: the high half of n m, and n itself, shifted (the quotient's multiplier has 33 bits, the highest of them set)
struct Divide {
  unsigned d, m, s;
  __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, m) + n) >> s; }
};
inline Divide divide_by(long long d) {
  unsigned s = 0;
  while ((1ll << s) < d) ++s;
  return Divide{(unsigned)d, (unsigned)((((1ull << s) - (unsigned long long)d) << 32) / (unsigned long long)d + 1), s};
}

}  // namespace mlstm
