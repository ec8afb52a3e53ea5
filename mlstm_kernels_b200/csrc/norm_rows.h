// How layer norm's kernels take a row of D elements (plain numbers: also for the host compiler).
#pragma once
#include <cstddef>

namespace mlstm {

constexpr int LN_V = 16;           // elements of a row to a thread
constexpr int LN_MAX_D = 16384;    // 1024 threads, twice eight elements

// Threads to a row: a power of two up to a warp, then as many warps as it takes up to 256 threads.  32768 rows in bf16, forward and
// backward's pass, against the next power of two: 96 threads (1104 elements) 33.2 and 70.8 us against 41.6 and 84.1; 160 (2304) 51.9 and
// 107 against 79.0 and 161; 192 (2904) 64.8 and 135 against 80.7 and 166; 224 (3304) 77.0 and 152 against 81.9 and 169.
inline int ln_threads(int D) {
  int t = 4;
  while (t < 32 && t * LN_V < D) t *= 2;
  if (t * LN_V < D) t = (D + 32 * LN_V - 1) / (32 * LN_V) * 32;
  return t <= 256 ? t : t <= 512 ? 512 : 1024;
}
// In chunks of 16 bytes, if rows are whole ones (and lie on such boundaries); a thread's chunks past the row's end stay empty, so the
// row need not fill all of them.
inline bool ln_whole_chunks(int D, size_t element_size) { return D * element_size % 16 == 0; }

}  // namespace mlstm
