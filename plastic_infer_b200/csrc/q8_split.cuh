// How the stream of units of the 8-bit decode attention is shared out, for the kernels and for a
// host-side check (tests/native/q8_split_check.cpp).
//
// The stream is every (request, head pass) segment's units one after another: request b's HV
// segments of uoff[b + 1] - uoff[b] units each begin at uoff[b] * HV. It is cut into equal ranges,
// one per active warp; a segment that a cut crosses is finished in pieces, one per warp over it.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define PI_HD __host__ __device__ __forceinline__
#else
#define PI_HD inline
#endif

namespace pi {
namespace q8 {

// Warps that share a stream of `total` units: every active warp owns at least one, two where there
// are enough (a piece more costs its merge more than a unit costs its warp: 1000 tokens of 8 KV
// heads take 14.6 us against 16.5 with one unit per warp).
PI_HD int active_warps(int64_t total, int nw) {
  const int64_t most = (total + 1) / 2;
  return static_cast<int>(most < nw ? most : nw);
}

struct Split {
  int64_t total;
  int warps;
  PI_HD int64_t first(int w) const { return total * w / warps; }  // of warp w's range
  PI_HD int owner(int64_t pos) const { return static_cast<int>(((pos + 1) * warps - 1) / total); }
};

// Request of stream position pos.
PI_HD int request_at(const int* uoff, int requests, int HV, int64_t pos) {
  int l = 0, r = requests - 1;
  while (l < r) {
    const int mid = (l + r + 1) >> 1;
    if (static_cast<int64_t>(uoff[mid]) * HV <= pos) l = mid; else r = mid - 1;
  }
  return l;
}

// A warp that gives up at position pos of its range still arrives at every cut segment that it has not
// finished, so that the segments' counters come back to zero (their outputs are unspecified then).
// arrive(segment, pieces) counts one arrival of `pieces`.
template <typename Arrive>
PI_HD void abandon(const Split& s, const int* uoff, int requests, int HV, int warp, int64_t pos, Arrive arrive) {
  const int64_t lo = s.first(warp), hi = s.first(warp + 1);
  while (pos < hi) {
    const int b = request_at(uoff, requests, HV, pos);
    const int64_t first = static_cast<int64_t>(uoff[b]) * HV;
    const int n = uoff[b + 1] - uoff[b];
    const int hv = static_cast<int>((pos - first) / n);
    const int64_t start = first + static_cast<int64_t>(hv) * n, end = start + n;
    if (start < lo || end > hi) arrive(b * HV + hv, s.owner(end - 1) - s.owner(start) + 1);
    pos = end;
  }
}

}  // namespace q8
}  // namespace pi
