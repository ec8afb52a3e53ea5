// How a gated linear recurrence is cut into units of work (plain numbers: also for the host compiler).
#pragma once
#include <algorithm>
#include <cstddef>

namespace mlstm {

constexpr int GATED_CK = 8;      // tokens to a thread, and to a state that the forward keeps for the backward
constexpr int GATED_CHANNELS = 64;   // of a unit
constexpr int GATED_WARPS = 7;   // most warps of a CTA that take tokens; one more hands the states on
constexpr int GATED_GROUP = 16;  // most units of a group

// A unit is `warps` * GATED_CK tokens of GATED_CHANNELS channels of one sequence (a chain).  Units are numbered by time, the chains of one
// time after one another, and taken in that order.  `group` units of a chain that follow one another take the state in front of their
// group and join what stands between by themselves.
struct GatedPlan {
  int blocks, warps, nt, group, groups;   // units beside each other in D, warps of a CTA, units and groups of a chain
  long long chains, units;
};
inline GatedPlan gated_plan(int B, int S, int D, int slots) {
  GatedPlan p{};
  const int runs = (S + GATED_CK - 1) / GATED_CK;
  p.blocks = (D + GATED_CHANNELS - 1) / GATED_CHANNELS;
  p.nt = (runs + GATED_WARPS - 1) / GATED_WARPS;
  p.warps = (runs + p.nt - 1) / p.nt;
  p.chains = (long long)B * p.blocks;
  p.units = p.chains * p.nt;
  // As long as a unit's predecessors in its chain are under way beside it, groups are what keeps them from waiting for one another:
  // 1 x 65536 x 2048 takes 1117, 742, 641, 606, 553 us with groups of 1, 2, 4, 8, 16, 1 x 65536 x 64 892 with 1, 75 with 16 (and 61
  // with 32, which every unit of a group would join up to 31 runs for).  Where there are more chains than CTAs a group is two units.
  const long long beside = (slots + p.chains - 1) / p.chains;
  p.group = 1;
  while (p.group < GATED_GROUP && p.group < beside * 2 && p.group < p.nt) p.group *= 2;
  p.groups = (p.nt + p.group - 1) / p.group;
  return p;
}

// Scratch, offsets in bytes: a counter, states in front of groups and runs of units, all of which a call zeroes first (none where a
// chain is one unit), and sums of the rate's gradient (backward).
struct GatedScratch { size_t state, agg, rate, bytes; };
inline size_t gated_up(size_t n) { return (n + 255) / 256 * 256; }
inline GatedScratch gated_scratch(const GatedPlan& p, int B, int D, bool backward) {
  GatedScratch s{};
  s.state = p.nt > 1 ? 256 : 0;
  s.agg = s.state + (p.nt > 1 ? gated_up(32 * 8 * (size_t)p.chains * p.groups) : 0);
  s.rate = s.agg + (p.group > 1 ? gated_up(32 * 16 * (size_t)p.units) : 0);
  s.bytes = s.rate + (backward ? gated_up(4 * (size_t)B * p.nt * D) : 0);
  return s;
}

}  // namespace mlstm
