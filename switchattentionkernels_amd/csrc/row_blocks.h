// Listed query rows and the key tiles that they see: what the backward and the
// sums of attention weights have in common.  Rows are ordered as in the forward
// (compacted query slot, head of the group; head fastest), in blocks.  Templates
// over the kernels' parameters P: the lists (idx, count), the bounds (starts,
// ends; kMeta) or the shape they follow from (seq_q, seq_kv, window), total_q,
// total_kv, group, and the ranges to fill.
#pragma once

#include "common.h"

namespace swattn {
namespace {

// A listed position outside [0, total_q) is never dereferenced: the host
// checks the lists before the launch, and this keeps a list changed after
// that check from turning into an out-of-bounds access.
template <class P>
__device__ __forceinline__ bool pos_ok(const P& p, int pos) {
  return static_cast<uint32_t>(pos) < static_cast<uint32_t>(p.total_q);
}

template <bool kMeta, class P>
__device__ __forceinline__ void row_bounds(const P& p, int branch, int pos, int& ks,
                                           int& ke) {
  if constexpr (kMeta) {
    ks = p.starts[branch][pos];
    ke = p.ends[pos];
  } else {
    const int b = pos / p.seq_q;
    const int i = pos - b * p.seq_q;
    const int base = b * p.seq_kv;
    ke = base + min(i + 1, p.seq_kv);
    ks = branch == 0 ? base : base + max(i - p.window + 1, 0);
  }
  ks = max(ks, 0);
  ke = min(ke, p.total_kv);
  // An empty range keeps ks = ke.  F's rule with seq_q > seq_kv + window - 1
  // gives late local rows a start past their end (and past the next
  // sequence's first start); clipped, the starts are non-decreasing along
  // each list, as the search of block_ranges needs.
  ks = min(ks, ke);
}

// ---------------------------------------------------------------------------
// Block ranges: for each branch and tile of kKeys keys, the blocks of kRows rows whose
// rows can see a key of the tile.  Row bounds are non-decreasing along each
// list, so the slots that overlap [k0, k1) are [first with end > k0, first
// with start >= k1).
// ---------------------------------------------------------------------------
// The first slot in [lo, hi) of list b whose row bounds satisfy pred (false
// ... false, true ... true along the list), or hi.  A wave searches
// together: each step probes 64 evenly spaced slots at once and keeps the
// gap between the last false and the first true probe, so a list of n slots
// costs about log64(n) dependent loads instead of log2(n).  lo and hi stay
// wave-uniform (ballot), and every probe lies in [lo, hi).
template <bool kMeta, class P, class Pred>
__device__ int wave_lower_bound(const P& p, int b, int lo, int hi, Pred pred) {
  const int lane = threadIdx.x & 63;
  while (lo < hi) {
    const int64_t span = hi - lo;
    const int probe = lo + static_cast<int>(span * lane / 64);
    const int pm = p.idx[b][probe];
    int ks, ke;
    row_bounds<kMeta>(p, b, pos_ok(p, pm) ? pm : 0, ks, ke);
    const uint64_t m = __builtin_amdgcn_ballot_w64(pred(ks, ke));
    if (m == 0) {
      lo += static_cast<int>(span * 63 / 64) + 1;   // past the last probe
    } else {
      const int first = __builtin_ctzll(m);
      hi = lo + static_cast<int>(span * first / 64);
      if (first > 0) lo += static_cast<int>(span * (first - 1) / 64) + 1;
    }
  }
  return lo;
}

// One wave per (branch, key tile); workgroups of 256 threads.
template <bool kMeta, int kKeys, int kRows, class P>
__device__ __forceinline__ void block_ranges(const P& p, int tiles, int wg) {
  const int i = (wg * 256 + threadIdx.x) >> 6;
  if (i >= 2 * tiles) return;   // whole waves
  const int b = i / tiles, t = i - b * tiles;
  const int k0 = t * kKeys, k1 = min(k0 + kKeys, p.total_kv);
  const int n = p.count[b];
  const int s_lo = wave_lower_bound<kMeta>(p, b, 0, n, [=](int, int ke) { return ke > k0; });
  const int s_hi = wave_lower_bound<kMeta>(p, b, s_lo, n, [=](int ks, int) { return ks >= k1; });
  int blo = 0, bhi = 0;
  if (s_lo < s_hi) {
    const int64_t G = p.group;
    blo = static_cast<int>((s_lo * G) / kRows);
    bhi = static_cast<int>((s_hi * G + kRows - 1) / kRows);
  }
  if ((threadIdx.x & 63) == 0) {
    p.ranges[2 * i] = blo;
    p.ranges[2 * i + 1] = bhi;
  }
}

}  // namespace
}  // namespace swattn
