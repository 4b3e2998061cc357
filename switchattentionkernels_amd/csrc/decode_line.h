// The line of routed keys that a decode call shares out over the chip's
// workgroups, and the merge of the workgroups' partial results: what the decode
// over bf16 caches and the one over 8-bit caches have in common.  Templates over
// the kernels' parameters P, a DecodeCommon with the shares' constants and
// kKeepNan: whether a partial whose sum is NaN makes the row NaN (false: it is
// left out of the row).
#pragma once

#include <math.h>

#include "common.h"

namespace swattn {
namespace {

constexpr int kD = 128;
constexpr int kMaxSplitsDev = 256;   // partials per (sequence, KV head), at most
constexpr int kInlinePer = 4;        // sequences per thread that a split workgroup plans itself
constexpr int kInlineSeqs = 256 * kInlinePer;

struct DecodeCommon {
  const int32_t* lens;
  const uint8_t* full;
  float* part_o;     // [slot][G][128] unnormalised sum of p * v, per workgroup and pair
  float* part_ml;    // [slot][G][2]   maximum (exp2 domain) and sum of p
  int32_t* list;     // sequences with keys, in order                      (plan kernel)
  uint4* plan;       // [0] {positions per workgroup, positions of the line (low, high)}; [1 + b]
                     // plan_entry of sequence b
  uint16_t* out;
  float* lse;
  int cache_len;     // L
  int batch, hq, hkv, group, window;
  uint32_t target;   // workgroups that are resident at once
  uint32_t pad;      // line positions a pair takes beside its keys (shared layout)
};

// Key range of sequence b: first key and number of keys.
template <class P>
__device__ __forceinline__ void key_range(const P& p, int b, int& lo, int& n) {
  const int len = min(max(p.lens[b], 0), p.cache_len);
  lo = p.full[b] ? 0 : max(len - p.window, 0);
  n = len - lo;
}

// The line's layout, chosen from the total of routed keys and the number of
// pairs that have any (both over all KV heads).  Positions are 32-bit where the
// workgroups plan for themselves, which they do for caches of fewer than 2^31
// rows (512 GiB), and 64-bit in the plan kernel; a share and a pair's keys fit 32
// bits in both (the host sees to it).
//
// * Shared: every pair takes its keys plus p.pad positions (what starting a
//   pair costs, in keys), and the line is cut into p.target equal shares,
//   twice as many when a share is long (kLongShare: two rounds then even out
//   the CUs' speeds).  B64 L4096-8192 Hq32/Hkv8 p_full 0.25: 144.5 us without
//   padding, 142.3 with 64 positions, 139.1 with 192, 139.9 with 256; B40
//   L2500-5000 Hq64/Hkv8 W512: 78.7 with 64, 72.5 with 192; all full, B64:
//   321 us with shares of 6144 keys left whole, 310 halved.
// * Aligned, for few pairs: every pair takes a whole number of shares, so that
//   no workgroup takes pieces of two pairs one after the other (about 4 us).
//   p.target shares then hold every pair if each is total / (p.target - pairs)
//   keys long; taken while that is at most kAlignSlack keys more than the
//   shared layout's, less time than the second piece's start.  One cache of
//   about 3300 keys, Hq32/Hkv8: 14.6 us, shared 18.9; B8 L2048-4096 p_full
//   0.5: 28.6 against 31.5.
//
// A share is at least kMinShare keys and at least ceil(L / 255), so that a
// pair is spread over at most 256 workgroups, rounded up to 16.
template <typename Pos>
struct Line {
  uint32_t share, aligned;
  Pos total;   // positions of the line
  __device__ __forceinline__ uint32_t length(uint32_t n, uint32_t pad) const {
    return n == 0 ? 0u : aligned ? (n + share - 1u) / share * share : n + pad;
  }
};
template <typename Pos, class P>
__device__ __forceinline__ Line<Pos> plan_line(const P& p, Pos keys, uint32_t pairs) {
  const uint32_t target = p.target;
  const uint32_t by_len = (static_cast<uint32_t>(p.cache_len) + kMaxSplitsDev - 2u) / (kMaxSplitsDev - 1u);
  const uint32_t least = max(by_len, P::kMinShare);
  Line<Pos> L;
  L.total = keys + pairs * p.pad;
  L.share = static_cast<uint32_t>((L.total + target - 1u) / target);
  L.aligned = 0u;
  if (pairs < target) {
    const Pos a = max((keys + target - pairs - 1u) / (target - pairs), static_cast<Pos>(least));
    if (a <= max(L.share, least) + P::kAlignSlack) {
      L.aligned = 1u;
      L.share = static_cast<uint32_t>(a);
    }
  }
  if (L.aligned == 0u && L.share >= P::kLongShare) L.share = (L.share + 1u) / 2u;
  L.share = (max(L.share, least) + 15u) & ~15u;
  return L;
}

// Exclusive prefix sums over the workgroup's threads of (keys, cnt), and both
// totals; one barrier.  (kUse: calls of one kernel use separate LDS words.)
template <int kWaves, int kUse, typename Pos>
__device__ __forceinline__ void scan_keys(Pos keys, uint32_t cnt, Pos& keys_before,
                                          uint32_t& cnt_before, Pos& keys_total,
                                          uint32_t& cnt_total) {
  __shared__ Pos s_keys[kWaves];
  __shared__ uint32_t s_cnt[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Pos ik = keys;
  const uint32_t ic = wave_sums(cnt);
  if constexpr (sizeof(Pos) == 4) {
    ik = wave_sums(keys);
  } else {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const Pos uk = __shfl_up(ik, off);
      ik += lane >= off ? uk : Pos{0};
    }
  }
  if (lane == 63) {
    s_keys[wave] = ik;
    s_cnt[wave] = ic;
  }
  __syncthreads();
  keys_before = ik - keys;
  cnt_before = ic - cnt;
  keys_total = Pos{0};
  cnt_total = 0u;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    keys_before += w < wave ? s_keys[w] : Pos{0};
    cnt_before += w < wave ? s_cnt[w] : 0u;
    keys_total += s_keys[w];
    cnt_total += s_cnt[w];
  }
}

// Sequence b's place on the line as the merge (and the listed plan) reads it:
// position of its first key, its keys, its rank among those with keys, positions
// per pair.  Ranks are below 65536, so the position has 48 bits.
struct SeqPlace {
  uint64_t off;
  uint32_t n, rank, len;
};
__device__ __forceinline__ uint4 plan_entry(uint64_t off, uint32_t n, uint32_t rank, uint32_t len) {
  return make_uint4(static_cast<uint32_t>(off), n, rank | static_cast<uint32_t>(off >> 32) << 16, len);
}
__device__ __forceinline__ SeqPlace seq_place(const uint4& e) {
  return SeqPlace{e.x | static_cast<uint64_t>(e.z >> 16) << 32, e.y, e.z & 0xffffu, e.w};
}

// a / b where the quotient fits 32 bits.
__device__ __forceinline__ uint32_t quotient(uint64_t a, uint32_t b) {
  return (a >> 32) == 0 ? static_cast<uint32_t>(a) / b : static_cast<uint32_t>(a / b);
}

// A sequence with keys: its index, first key, number of keys, and the
// positions each of its pairs takes on the line.
struct SeqEntry {
  int b, lo, n;
  uint32_t len;
};

// Where a split workgroup starts on the line: position `key` of pair (entry r,
// KV head kvh), and how many positions it takes.
struct SplitStart {
  uint32_t r, kvh, key, take;
};

// Start inside the sequence of rank r, from_off positions after its first; its
// pairs take len positions each.
__device__ __forceinline__ void split_start(SplitStart& st, uint32_t r, uint64_t from_off,
                                            uint32_t len) {
  st.r = r;
  st.kvh = quotient(from_off, len);
  st.key = static_cast<uint32_t>(from_off - static_cast<uint64_t>(st.kvh) * len);
}

// The start of this workgroup, found by itself: thread t holds sequences
// per*t .. per*t + per - 1 (per = ceil(batch / 256), at most kInlinePer), the
// workgroup scans their routed keys, keeps the sequences that have any in LDS
// and the one thread whose sequences hold line position blockIdx.x * share
// publishes it.  The lengths and routes are L2-resident after the first
// workgroups; against a list planned by a kernel of its own this costs about
// the same dependent latency and saves the launch (5-7 us of a 24-150 us
// call).  Workgroup 0 leaves every sequence's place on the line for the merge.
// Returns false past the end of the line.
template <class P>
__device__ __forceinline__ bool plan_inline(const P& p, SeqEntry* s_ent, SplitStart& st) {
  __shared__ SplitStart s_start;
  const int tid = threadIdx.x;
  const int per = (p.batch + 255) >> 8;
  int lo[kInlinePer], n[kInlinePer];
  uint32_t keys = 0, cnt = 0;
#pragma unroll
  for (int j = 0; j < kInlinePer; ++j) {
    const int b = tid * per + j;
    lo[j] = n[j] = 0;
    if (j < per && b < p.batch) key_range(p, b, lo[j], n[j]);
    keys += n[j];
    cnt += n[j] > 0 ? 1 : 0;
  }
  uint32_t before, rank, all_keys, all_cnt;
  scan_keys<4, 0, uint32_t>(keys, cnt, before, rank, all_keys, all_cnt);
  Line<uint32_t> L = plan_line<uint32_t>(p, all_keys * p.hkv, all_cnt * p.hkv);
  before += rank * p.pad;
  if (L.aligned) {
    uint32_t len = 0, none;
#pragma unroll
    for (int j = 0; j < kInlinePer; ++j) len += L.length(n[j], 0);
    scan_keys<4, 1, uint32_t>(len, 0, before, none, L.total, none);
    L.total *= p.hkv;
  }
  const uint64_t pos64 = static_cast<uint64_t>(blockIdx.x) * L.share;
  const uint32_t pos = static_cast<uint32_t>(min(pos64, static_cast<uint64_t>(L.total)));
#pragma unroll
  for (int j = 0; j < kInlinePer; ++j) {
    const int b = tid * per + j;
    const uint32_t off = before * p.hkv, len = L.length(n[j], p.pad);
    if (blockIdx.x == 0 && j < per && b < p.batch) p.plan[1 + b] = plan_entry(off, n[j], rank, len);
    if (n[j] > 0) {
      s_ent[rank] = SeqEntry{b, lo[j], n[j], len};
      if (pos >= off && pos - off < len * p.hkv) split_start(s_start, rank, pos - off, len);
      ++rank;
    }
    before += len;
  }
  if (blockIdx.x == 0 && tid == 0) p.plan[0] = make_uint4(L.share, L.total, 0u, 0u);
  if (pos >= L.total) return false;   // uniform
  __syncthreads();
  st = s_start;
  st.take = min(L.total - pos, L.share);
  return true;
}

// The sequences' places on the line for more of them than that: one workgroup
// of 1024 threads.
constexpr int kPlanThreads = 1024;
template <class P>
__global__ __launch_bounds__(kPlanThreads) void decode_plan_kernel(const P p) {
  const int tid = threadIdx.x;
  const int per = (p.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  uint64_t keys = 0;
  uint32_t cnt = 0;
  for (int b = b0; b < b1; ++b) {
    int lo, n;
    key_range(p, b, lo, n);
    keys += n;
    cnt += n > 0 ? 1 : 0;
  }
  uint64_t before, all_keys;
  uint32_t rank, all_cnt;
  scan_keys<kPlanThreads / 64, 0, uint64_t>(keys, cnt, before, rank, all_keys, all_cnt);
  Line<uint64_t> L = plan_line<uint64_t>(p, all_keys * p.hkv, all_cnt * p.hkv);
  before += static_cast<uint64_t>(rank) * p.pad;
  if (L.aligned) {   // few of the sequences hold keys
    uint64_t len = 0;
    uint32_t none;
    for (int b = b0; b < b1; ++b) {
      int lo, n;
      key_range(p, b, lo, n);
      len += L.length(n, 0);
    }
    scan_keys<kPlanThreads / 64, 1, uint64_t>(len, 0, before, none, L.total, none);
    L.total *= p.hkv;
  }
  for (int b = b0; b < b1; ++b) {
    int lo, n;
    key_range(p, b, lo, n);
    const uint32_t len = L.length(n, p.pad);
    p.plan[1 + b] = plan_entry(before * p.hkv, n, rank, len);
    if (n > 0) p.list[rank++] = b;
    before += len;
  }
  if (tid == 0) p.plan[0] = make_uint4(L.share, static_cast<uint32_t>(L.total), static_cast<uint32_t>(L.total >> 32), 0u);
}

// The start of this workgroup from the plan kernel's table: a search for the
// last sequence whose line position is at or before the workgroup's (one with
// keys: the sequences after it start later, and one without keys shares its
// position with the next).  Every thread runs the same search.
template <class P>
__device__ __forceinline__ bool plan_listed(const P& p, SplitStart& st) {
  const uint4 line = p.plan[0];
  const uint32_t share = line.x;
  const uint64_t total = line.y | static_cast<uint64_t>(line.z) << 32;
  const uint64_t pos = static_cast<uint64_t>(blockIdx.x) * share;
  if (pos >= total) return false;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (seq_place(p.plan[1 + mid]).off <= pos) lo = mid; else hi = mid - 1;
  }
  const SeqPlace q = seq_place(p.plan[1 + lo]);
  split_start(st, q.rank, pos - q.off, q.len);
  st.take = static_cast<uint32_t>(min(total - pos, static_cast<uint64_t>(share)));
  return true;
}

// One workgroup of 256 threads per output row (b, head): merge the split partials.  Thread
// (g, q) = (tid / 32, tid % 32) takes dims 4q .. +3 of splits g, g + 8, ...;
// the first kMergeAhead of them are loaded before the weights are known, so
// that a row of up to 32 splits costs one memory latency.  Latency-bound:
// each row reads its splits' 512-byte rows once.
constexpr int kMergeAhead = 4;
template <class P>
__device__ __forceinline__ void merge_row(const P& p, int64_t row) {
  __shared__ float s_w[kMaxSplitsDev];
  __shared__ float s_red[8];
  __shared__ float4 s_part[8][kD / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = static_cast<int>(row / p.hq), hq = static_cast<int>(row - static_cast<int64_t>(b) * p.hq);
  const int kvh = hq / p.group, h = hq - kvh * p.group;
  // The pair's place on the line, the workgroups that share it and its slots.
  const SeqPlace seq = seq_place(p.plan[1 + b]);
  const uint32_t share = p.plan[0].x;
  const uint64_t off = seq.off + static_cast<uint64_t>(kvh) * seq.len;
  const uint32_t wg0 = quotient(off, share);
  const int nch = seq.n > 0 ? static_cast<int>(quotient(off + seq.n - 1, share) - wg0) + 1 : 0;   // at most 256
  const int64_t slot0 = static_cast<int64_t>(wg0) + static_cast<int64_t>(seq.rank) * p.hkv + kvh;
  const int g = tid >> 5, q = tid & 31;
  const float4* base = reinterpret_cast<const float4*>(p.part_o + (slot0 * p.group + h) * kD) + q;
  const int64_t cstride = static_cast<int64_t>(p.group) * (kD / 4);
  float2 ml = make_float2(-INFINITY, 0.f);   // split tid's maximum and sum
  if (tid < nch) ml = *reinterpret_cast<const float2*>(p.part_ml + ((slot0 + tid) * p.group + h) * 2);
  float4 ahead[kMergeAhead];
#pragma unroll
  for (int i = 0; i < kMergeAhead; ++i) {
    ahead[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g + 8 * i < nch) ahead[i] = base[(g + 8 * i) * cstride];
  }
  // Maximum over the non-empty splits.
  auto holds = [](float sum) { return P::kKeepNan ? sum != 0.f : sum > 0.f; };
  float mx = holds(ml.y) ? ml.x : -INFINITY;
  mx = wave_all(mx, Max());
  if (lane == 0) s_red[wave] = mx;
  __syncthreads();
  const float M = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  // Split weights 2^(m_c - M) (0 for empty splits) and the weighted sum of l.
  const float wt = (holds(ml.y) && M != -INFINITY) ? __builtin_amdgcn_exp2f(ml.x - M) : 0.f;
  s_w[tid] = wt;
  float lsum = wt * ml.y;
  lsum = wave_all(lsum, Add());
  if (lane == 0) s_red[4 + wave] = lsum;
  __syncthreads();
  const float L = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  // Weighted sum of the unnormalised partial outputs.
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int c, const float4& x) {
    const float w = s_w[c];
    if (P::kKeepNan || w != 0.f) {
      a.x += w * x.x;
      a.y += w * x.y;
      a.z += w * x.z;
      a.w += w * x.w;
    }
  };
#pragma unroll
  for (int i = 0; i < kMergeAhead; ++i)
    if (g + 8 * i < nch) add(g + 8 * i, ahead[i]);
#pragma unroll 4
  for (int c = g + 8 * kMergeAhead; c < nch; c += 8) add(c, base[c * cstride]);
  s_part[g][q] = a;
  __syncthreads();
  if (tid < kD) {
    const float* part = reinterpret_cast<const float*>(s_part) + tid;
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc += part[i * kD];
    const float o = acc / L;   // empty row: 0 / 0 = NaN, as the prefill writes it
    p.out[row * kD + tid] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(o));
    if (tid == 0) p.lse[row] = M == -INFINITY && !(P::kKeepNan && L != L) ? -INFINITY : M + log2f(L);
  }
}

}  // namespace
}  // namespace swattn
