// Host-side check of plastic_infer_b200/csrc/q8_split.cuh: over random batches, every segment's pieces
// are the warps that hold its units, counted unit by unit, and the arrival counters come back to zero
// when any of the warps give up at any unit of their ranges. Prints "ok" and exits 0.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "q8_split.cuh"

using namespace pi::q8;

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  long left_over = 0, cut = 0, gave_up = 0;
  for (int trial = 0; trial < 4000; ++trial) {
    const int B = pick(1, 12), HV = pick(1, 9), NW = pick(1, 80);
    std::vector<int> uoff(B + 1, 0);
    for (int b = 0; b < B; ++b) uoff[b + 1] = uoff[b] + (pick(0, 3) ? pick(0, 40) : 0);
    const int64_t total = static_cast<int64_t>(uoff[B]) * HV;
    if (total == 0) continue;
    const Split s{total, active_warps(total, NW)};
    // unit by unit: its segment, its warp
    std::vector<int> segment, warp;
    for (int b = 0; b < B; ++b)
      for (int h = 0; h < HV; ++h)
        for (int u = uoff[b]; u < uoff[b + 1]; ++u) segment.push_back(b * HV + h);
    for (int w = 0; w < s.warps; ++w)
      for (int64_t p = s.first(w); p < s.first(w + 1); ++p) warp.push_back(w);
    if (static_cast<int64_t>(warp.size()) != total || static_cast<int64_t>(segment.size()) != total) return std::puts("sizes"), 1;
    std::vector<int> pieces(B * HV, 0);
    for (int64_t p = 0; p < total; ++p) {
      if (s.owner(p) != warp[p]) return std::puts("owner"), 1;
      if (request_at(uoff.data(), B, HV, p) != segment[p] / HV) return std::puts("request"), 1;
      if (p == 0 || segment[p] != segment[p - 1] || warp[p] != warp[p - 1]) ++pieces[segment[p]];
    }
    // the warps one after another, in any order; a failing one stops at some unit of its range
    std::vector<int> order(s.warps), counter(B * HV, 0), without(B * HV, 0);
    for (int w = 0; w < s.warps; ++w) order[w] = w;
    std::shuffle(order.begin(), order.end(), rng);
    bool bad = false;
    auto arrive = [&](std::vector<int>& c, int seg, int n) {
      if (n != pieces[seg]) bad = true;
      if (++c[seg] == n) c[seg] = 0;
    };
    for (int w : order) {
      const int64_t lo = s.first(w), hi = s.first(w + 1);
      const int64_t stop = pick(0, 2) == 0 ? lo + pick(0, static_cast<int>(hi - lo) - 1) : hi;
      for (int64_t p = lo; p < stop; ++p) {  // a piece is finished at its last unit
        const int seg = segment[p];
        if (pieces[seg] > 1 && (p + 1 == hi || segment[p + 1] != seg)) {
          arrive(counter, seg, pieces[seg]);
          arrive(without, seg, pieces[seg]);
          ++cut;
        }
      }
      if (stop < hi) {
        ++gave_up;
        // stop is a unit that was not finished: its piece, and those after it, have not arrived
        abandon(s, uoff.data(), B, HV, w, stop, [&](int seg, int n) { arrive(counter, seg, n); });
      }
    }
    if (bad) return std::puts("pieces"), 1;
    for (int c : counter)
      if (c != 0) return std::puts("a counter is left over"), 1;
    for (int c : without) left_over += c;
  }
  if (cut == 0 || gave_up == 0 || left_over == 0) return std::puts("nothing was checked"), 1;
  std::puts("ok");
  return 0;
}
