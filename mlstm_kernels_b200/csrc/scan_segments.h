// Into how many segments the selective state space scan cuts a sequence (plain numbers: also for the host compiler).
#pragma once
#include <cmath>
#include <cstddef>

namespace mlstm {

// CTAs that an SM holds at once: of `bytes` of shared memory each (and 1 KB for the system, of 228 KB), at most `most`, by registers
constexpr int scan_resident(size_t bytes, int most) {
  const size_t n = 228 * 1024 / (bytes + 1024);
  return n < 1 ? 1 : n > (size_t)most ? most : (int)n;
}
struct ScanSlots { int whole, own; };   // of the pass over all segments, and of the one for their own ends

// The time of a launch of `grid` CTAs, up to `slots` to an SM, for each tile of a CTA: k of them share an SM for k + add, at least
// `alone`.  More than fit go round; the last round counts half as full as it is not.
inline float scan_rounds(long long grid, int slots, float add, float alone, int sms) {
  const float per_sm = (float)grid / (float)sms, rounds = per_sm / (float)slots;
  const float k = rounds > 1.f ? (float)slots : std::ceil(per_sm), tile = k + add > alone ? k + add : alone;
  return rounds > 1.f ? 0.5f * (rounds + std::ceil(rounds)) * tile : tile;
}

// The number that should take least, the pass over the segments' own ends (for all but one) and its launch among it.
// ctas: of a segment in the pass over all, `turns` tiles of channels each; own_ctas: in the other; nt: tiles of a sequence; np: states.
// Units of a tile's part of a full SM: 0.9 us forward, 4.1 us backward.  A tile takes a CTA alone 2.5 units forward (2.0-2.4 us with 8 to
// 32 states), with more states longer, as each CTA widens the tile's 32 np values of b and c: 3.2 us with 64, 4.7 with 128.
// Measured, bf16: 4 x 2048 x 2048 channels of 16 states forward 294, 210, 198, 193, 190 us with 1, 5, 8, 10, 16 segments, backward 1777,
// 703, 533, 567, 521; of 8 states 312, 233, 151, 149, 130 and 1130, 564, 394, 438, 369 (two CTAs of the backward to an SM; in f32 one:
// 958, 695, 611, 580, 536); 512 x 1024 channels of 16 states forward 68, 34, 23, 22 with 1, 4, 16, 32; of 128 states 152, 87, 85, 98 with
// 1, 4, 5, 16; 128 CTAs of 8 tiles: 20 and 24 with 1 and 4.
inline int scan_segments(long long ctas, int turns, long long own_ctas, int nt, int np, bool backward, ScanSlots slots, int sms) {
  const float alone = backward ? 4.f : np >= 128 ? 5.f : np >= 64 ? 3.5f : 0.f;
  int best = 1;
  float least = 0.f;
  for (int n = 1; n <= 64 && (n == 1 || n <= nt); ++n) {
    const int seg = (nt + n - 1) / n;
    if (n > 1 && (nt + seg - 1) / seg != n) continue;
    float t = (float)turns * scan_rounds(ctas * n, slots.whole, backward ? 0.f : 1.5f, alone, sms);
    if (n > 1) t += (backward ? 0.13f : 0.6f) * scan_rounds(own_ctas * (n - 1), slots.own, 1.5f, 0.f, sms);
    t *= (float)seg + 0.5f;                      // (half a tile's time to begin and to end)
    if (n > 1) t += backward ? 0.7f : 3.3f;      // 3 us
    if (n == 1 || t < least) { best = n; least = t; }
  }
  return best;
}

}  // namespace mlstm
