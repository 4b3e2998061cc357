// The 8-bit KV cache for gfx950: appending bf16 rows, reading rows back, and
// eviction by accumulated attention weight (include/swattn_cache.h).  No
// counterpart in the reference, which is prefill-only.
//
// A cached value is code * scale, one scale s per block of tokens and KV head:
//   s = the smallest 2^e >= 2^-100 with max |x| <= qmax * 2^e over the block,
//   code = round(x / s).
// A power of two makes x / s exact, so that a value is rounded once, costs e4m3
// nothing (its steps are relative) and int8 at most one bit, half a bit on
// average.
//
// All three are HBM-bound: a row of one head is 256 bytes in bf16 and 128 as
// codes, for K and for V.  Workgroups of 256 threads take one block of one head:
// threads 0-127 its K rows, 128-255 its V rows, 16 rows at a time, 8 threads of
// 16 values per row.

#include <limits.h>

#include <string.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "cache_code.h"
#include "swattn_internal.h"

namespace swattn {
namespace {

using namespace code;

constexpr int kD = 128;
constexpr int kRowsAtOnce = 16;   // rows that a workgroup's half takes at once
// Reads and evictions that move this much stream the codes that they read past the
// 256 MB memory-side cache, which then keeps what they write: moving 192 MB, 48 us kept
// and 54 streamed (evict), 31.8 and 35.5 (read); 256 MB 69 and 68 (evict); 280 MB 54.6
// and 48.4 (read); 437 MB 114 and 104 (evict); 512 MB 136 and 126.  Appends do not: new
// rows are in that cache as a rule, from the kernel that made them (128 MB of them, made
// and appended: 85 us, streamed 92).  Streamed stores: a third slower.
constexpr int64_t kStreamBytes = int64_t{224} << 20;

__device__ __forceinline__ float bf(uint32_t bits16) { return __uint_as_float(bits16 << 16); }

// Largest magnitude's bits over this half of the workgroup (threads 0-127 or
// 128-255): lane moves inside a wave, one exchange between the half's two.
__device__ __forceinline__ uint32_t half_max(uint32_t x) {
  __shared__ int s_max[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int v = static_cast<int>(x);   // no sign
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));    // neighbours
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));    // pairs
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));   // mirror image of 8
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false));   // and of 16 lanes
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(static_cast<int>(a[0]), static_cast<int>(a[1]));
  const auto c = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(static_cast<int>(c[0]), static_cast<int>(c[1]));
  if (lane == 0) s_max[wave] = v;
  __syncthreads();
  return static_cast<uint32_t>(max(s_max[wave & 2], s_max[(wave & 2) + 1]));
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
struct AppendParams {
  const uint16_t* src[2];    // new K, V rows
  const int32_t* cu;         // packed: offsets, else null (or HostOffsets)
  const int32_t* counts;     // padded: rows per sequence, or null
  const int32_t* lens;
  uint8_t* codes[2];
  float* scales[2];
  int32_t* lens_out;
  int64_t rows, total_rows;
  int cache_len, hkv, nblk, blocks;   // blocks: per sequence, at most
};

// Packed offsets as kernel arguments: no copy of them to the device.
struct HostOffsets {
  int32_t cu[SWATTN_CACHE_HOST_MAX_SEQS + 1];
};
struct NoOffsets {};

// One workgroup per (sequence, touched block, KV head).
template <int kCode, int kBlock, class Offsets>
__global__ __launch_bounds__(256) void append_kernel(const AppendParams p, const Offsets host) {
  constexpr int kIt = kBlock / kRowsAtOnce;
  const int h = blockIdx.x % p.hkv;
  const int rest = blockIdx.x / p.hkv;
  const int i = rest % p.blocks, b = rest / p.blocks;
  const int len = min(max(p.lens[b], 0), p.cache_len);
  // This sequence's new rows: src rows first .. first + count - 1.
  int64_t first = b * p.rows, count = p.rows;
  auto packed = [&](const int32_t* cu) {
    first = min(max(static_cast<int64_t>(cu[b]), int64_t{0}), p.total_rows);
    count = min(min(max(static_cast<int64_t>(cu[b + 1]), first), p.total_rows) - first, p.rows);
  };
  if constexpr (std::is_same<Offsets, HostOffsets>::value) {
    packed(host.cu);
  } else if (p.cu != nullptr) {
    packed(p.cu);
  } else if (p.counts != nullptr) {
    count = min(max(static_cast<int64_t>(p.counts[b]), int64_t{0}), p.rows);
  }
  const int end = static_cast<int>(min(len + count, static_cast<int64_t>(p.cache_len)));
  if (i == 0 && h == 0 && threadIdx.x == 0) p.lens_out[b] = end;
  const int jb = len / kBlock + i;
  // uniform; blocks are counted, for the rows of those behind the cache may pass 2^31
  if (end <= len || jb > (end - 1) / kBlock) return;
  const int r0 = jb * kBlock;          // the block's rows
  const int half = threadIdx.x >> 7, t = threadIdx.x & 127;
  const int sub = t >> 3, piece = t & 7;
  const uint16_t* src = p.src[half];
  uint4 raw[kIt][2];
  uint32_t amax = 0;
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const int r = r0 + it * kRowsAtOnce + sub;
    raw[it][0] = raw[it][1] = make_uint4(0, 0, 0, 0);
    if (r >= len && r < end) {
      const uint4* row = reinterpret_cast<const uint4*>(src + ((first + (r - len)) * p.hkv + h) * kD + piece * 16);
      raw[it][0] = row[0];
      raw[it][1] = row[1];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t w[4] = {raw[it][u].x, raw[it][u].y, raw[it][u].z, raw[it][u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = max(amax, max((w[j] << 16) & 0x7fffffffu, w[j] & 0x7fff0000u));
    }
  }
  amax = half_max(amax);
  float scale = scale_for<kCode>(amax);
  const bool begun = r0 < len;
  float* sp = p.scales[half] + (static_cast<int64_t>(b) * p.hkv + h) * p.nblk + jb;
  uint8_t* codes = p.codes[half] + (static_cast<int64_t>(b) * p.cache_len * p.hkv + h) * kD + piece * 16;
  const int64_t stride = static_cast<int64_t>(p.hkv) * kD;
  if (begun) {
    const float old = *sp;
    scale = old != old || old > scale ? old : scale;   // NaN stays NaN
    __syncthreads();   // every thread has read the scale
    if (old == old && scale != old) {   // grown (or NaN now): round the held rows again
      const float ratio = old / scale;
#pragma unroll
      for (int it = 0; it < kIt; ++it) {
        const int r = r0 + it * kRowsAtOnce + sub;
        if (r < len) {
          uint4* at = reinterpret_cast<uint4*>(codes + r * stride);
          float x[16];
          decode16<kCode>(*at, x);
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] *= ratio;
          keep_finite<kCode>(scale, x);
          *at = encode16<kCode>(x);
        }
      }
    }
  }
  if (t == 0) *sp = scale;
  const float inv = 1.0f / scale;   // exact unless the scale is a begun block's own
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const int r = r0 + it * kRowsAtOnce + sub;
    if (r >= len && r < end) {
      float x[16];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t w[4] = {raw[it][u].x, raw[it][u].y, raw[it][u].z, raw[it][u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[8 * u + 2 * j] = bf(w[j] & 0xffffu);
          x[8 * u + 2 * j + 1] = bf(w[j] >> 16);
        }
      }
      if (begun) {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = x[j] / scale;
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= inv;
      }
      keep_finite<kCode>(scale, x);
      *reinterpret_cast<uint4*>(codes + r * stride) = encode16<kCode>(x);
    }
  }
}

// ---------------------------------------------------------------------------
// Read
// ---------------------------------------------------------------------------
struct ReadParams {
  const uint8_t* codes[2];
  const float* scales[2];
  const int32_t* starts;   // or null: `start`
  const int32_t* lens;     // or null: cache_len
  uint16_t* out[2];
  int64_t start;
  int32_t pieces;          // 16 values each, of one sequence's K
  int cache_len, hkv, nblk, block_log;
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<__bf16>(a))) |
         static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<__bf16>(b))) << 16;
}

// One thread per 16 values; blockIdx.y: sequence, blockIdx.z 0: K, 1: V.
template <int kCode, bool kStream>
__global__ __launch_bounds__(256) void read_kernel(const ReadParams p) {
  const uint32_t x = blockIdx.x * 256u + threadIdx.x;
  if (x >= static_cast<uint32_t>(p.pieces)) return;
  const int64_t b = blockIdx.y;
  const int which = blockIdx.z;
  const int piece = static_cast<int>(x & 7u);
  const uint32_t rowh = x >> 3, i = rowh / static_cast<uint32_t>(p.hkv);   // i * hkv + h
  const int h = static_cast<int>(rowh - i * static_cast<uint32_t>(p.hkv));
  const int64_t r = (p.starts != nullptr ? static_cast<int64_t>(p.starts[b]) : p.start) + i;
  const int end = p.lens != nullptr ? min(p.lens[b], p.cache_len) : p.cache_len;
  uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (r >= 0 && r < end) {
    const uint4 u = load_bytes<kStream, u32x4, uint4>(p.codes[which] + ((b * p.cache_len + r) * p.hkv + h) * kD + piece * 16);
    const float s = p.scales[which][(b * p.hkv + h) * p.nblk + (r >> p.block_log)];
    float v[16];
    decode16<kCode>(u, v);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      o[j] = make_uint4(pack_bf16(v[8 * j] * s, v[8 * j + 1] * s), pack_bf16(v[8 * j + 2] * s, v[8 * j + 3] * s),
                        pack_bf16(v[8 * j + 4] * s, v[8 * j + 5] * s), pack_bf16(v[8 * j + 6] * s, v[8 * j + 7] * s));
  }
  uint4* out = reinterpret_cast<uint4*>(p.out[which] + (b * p.pieces + x) * 16);
  out[0] = o[0];
  out[1] = o[1];
}

// ---------------------------------------------------------------------------
// Evict
// ---------------------------------------------------------------------------
struct EvictParams {
  const uint8_t* codes[2];
  const float* scales[2];
  const float* weights;
  const int32_t* lens;
  uint8_t* out_codes[2];
  float* out_scales[2];
  float* out_weights;
  int32_t* lens_out;
  int32_t* kept;   // [pair][budget - recent] rows that were chosen, ascending
  int cache_len, out_len, hkv, nblk, out_nblk, budget, recent;
};

// A weight as an unsigned number of the same order: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  if (w != w) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Which of the older rows stay: one workgroup per (sequence, KV head).  A radix
// search finds the (budget - recent)-th largest weight, 11, 11 and 10 bits at a
// time (the first digit holds the exponent and two mantissa bits, which spreads
// attention sums over many bins); one ordered pass then writes the rows above it
// and the first of those equal to it.  Wave w holds a run of consecutive rows, 64
// per step, so that ballots count and place them and the waves meet only once.
// kPer > 0: a thread's kPer weights are read once, into registers; 0: any number,
// read again in every pass.  Bound by latency: few workgroups for few sequences.
// 16384 rows, 8 pairs: 26 us with 8-bit digits and five reads, 12 so, 9.7 since a search
// ends where a whole bin stays, mostly after two digits.  Rows behind a sequence's end (key
// 0) stay out of the bins: all in one bin they took 17.5 us for 5000 rows where 7.0 do.
constexpr int kDigits = 2048;
constexpr int kSelectThreads = 1024;
template <int kThreads, int kPer>
__global__ __launch_bounds__(kThreads) void select_kernel(const EvictParams p) {
  constexpr int kWaves = kThreads / 64;
  constexpr int kBins = kDigits / kThreads;   // per thread
  __shared__ uint32_t s_hist[kDigits];
  __shared__ uint32_t s_wave[kWaves];
  __shared__ uint32_t s_pick[3];
  __shared__ uint2 s_count[kWaves];
  const int64_t pair = blockIdx.x;
  const int b = static_cast<int>(pair / p.hkv);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* w = p.weights + pair * p.cache_len;
#pragma unroll
  for (int i = 0; i < kBins; ++i) s_hist[tid + kThreads * i] = 0;
  // The weights do not wait for the length: all rows of the cache may be read.
  float ahead[kPer > 0 ? kPer : 1];
  if constexpr (kPer > 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) ahead[j] = w[min((wave * kPer + j) * 64 + lane, p.cache_len - 1)];
  }
  const int len = min(max(p.lens[b], 0), p.cache_len);
  if (pair - static_cast<int64_t>(b) * p.hkv == 0 && tid == 0) p.lens_out[b] = min(len, p.budget);
  const int want = p.budget - p.recent;
  if (len <= p.budget || want == 0) return;   // uniform
  const int n = len - p.recent;               // more than want
  const int steps = kPer > 0 ? kPer : (n + kThreads - 1) / kThreads;
  const int64_t first = static_cast<int64_t>(wave) * steps * 64 + lane;   // this thread's rows: first + 64 j
  // Key 0 for rows past the end: below every weight's.
  auto key_of = [&](int64_t i, float x) { return i < n ? order_key(x) : 0u; };
  uint32_t held[kPer > 0 ? kPer : 1];
  if constexpr (kPer > 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) held[j] = key_of(first + 64 * j, ahead[j]);
  }
  // f(row, key) for each of this thread's rows, in order.
  auto each = [&](auto&& f) {
    if constexpr (kPer > 0) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) f(first + 64 * j, held[j]);
    } else {
      for (int j = 0; j < steps; ++j) {
        const int64_t i = first + 64 * j;
        f(i, key_of(i, w[min(i, static_cast<int64_t>(n - 1))]));
      }
    }
  };
  uint32_t prefix = 0, mask = 0, need = want;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
    __syncthreads();   // the bins are clear
    each([&](int64_t, uint32_t k) {
      if (pass == 0 ? k != 0u : (k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & digits], 1u);
    });
    __syncthreads();
    // Bins from the top, kBins per thread; the one that holds the need-th key.
    uint32_t c[kBins], sum = 0;
#pragma unroll
    for (int j = 0; j < kBins; ++j) {
      uint32_t& bin = s_hist[kDigits - 1 - kBins * tid - j];
      c[j] = bin;
      bin = 0;   // for the next digit
      sum += c[j];
    }
    uint32_t incl = wave_sums(sum);
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kWaves; ++x) incl += x < wave ? s_wave[x] : 0u;
    uint32_t above = incl - sum;
    if (above < need && need <= incl) {   // one thread: the sums ascend
#pragma unroll
      for (int j = 0; j < kBins; ++j) {
        if (above < need && need <= above + c[j]) {
          s_pick[0] = kDigits - 1 - kBins * tid - j;
          s_pick[1] = need - above;
          s_pick[2] = c[j];
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    mask |= digits << shift;
    need = s_pick[1];
    if (need == s_pick[2]) break;   // uniform: all of the bin stay, whatever their other digits
  }
  // All rows above prefix stay, and the first `need` of those equal to it.
  int32_t* kept = p.kept + pair * want;
  if (need == s_pick[2]) {   // uniform: all of them
    uint32_t before = 0;
    each([&](int64_t, uint32_t k) { before += __builtin_popcountll(wave_ballot(k >= prefix)); });
    if (lane == 0) s_count[wave] = make_uint2(before, 0u);
    __syncthreads();
    before = 0;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) before += x < wave ? s_count[x].x : 0u;
    each([&](int64_t i, uint32_t k) {
      const uint64_t m = wave_ballot(k >= prefix);
      const uint32_t at = before + count_below(m);
      if (k >= prefix && at < static_cast<uint32_t>(want)) kept[at] = static_cast<int32_t>(i);
      before += __builtin_popcountll(m);
    });
    return;
  }
  uint32_t above = 0, equal = 0;
  each([&](int64_t, uint32_t k) {
    above += __builtin_popcountll(wave_ballot(k > prefix));
    equal += __builtin_popcountll(wave_ballot(k == prefix));
  });
  if (lane == 0) s_count[wave] = make_uint2(above, equal);
  __syncthreads();
  above = equal = 0;
#pragma unroll
  for (int x = 0; x < kWaves; ++x) {
    above += x < wave ? s_count[x].x : 0u;
    equal += x < wave ? s_count[x].y : 0u;
  }
  each([&](int64_t i, uint32_t k) {
    const uint64_t gt = wave_ballot(k > prefix), eq = wave_ballot(k == prefix);
    const uint32_t e = equal + count_below(eq);
    const uint32_t at = above + count_below(gt) + min(e, need);
    if ((k > prefix || (k == prefix && e < need)) && at < static_cast<uint32_t>(want))
      kept[at] = static_cast<int32_t>(i);
    above += __builtin_popcountll(gt);
    equal += __builtin_popcountll(eq);
  });
}

// The kept rows into the destination: one workgroup per (sequence, destination
// block, KV head).  32 sequences of 1024 to 4096 rows cut to 2047, 8 KV heads,
// blocks of 32, then read back: 146.5 us for search, copy and read, 144 since the chosen
// rows' loads do not wait for the length's, 136 streamed; the copy alone moves scattered
// 128-byte rows at 3.8 (traced) to 4.2 TB/s.  (64 rows a workgroup and a block's heads on one XCD were
// slower: 59 us, 64 and 62 when the copy took that.)
template <int kCode, int kBlock, bool kStream>
__global__ __launch_bounds__(256) void gather_kernel(const EvictParams p) {
  constexpr int kIt = kBlock / kRowsAtOnce;
  const int h = blockIdx.x % p.hkv;
  const int rest = blockIdx.x / p.hkv;
  const int jb = rest % p.out_nblk, b = rest / p.out_nblk;
  const int64_t pair = static_cast<int64_t>(b) * p.hkv + h;
  const int want = p.budget - p.recent;
  const int r0 = jb * kBlock;
  const int half = threadIdx.x >> 7, t = threadIdx.x & 127;
  const int sub = t >> 3, piece = t & 7;
  // The chosen rows do not wait for the length (which may leave them unused).
  const int32_t* kept = p.kept + pair * want;
  int chosen[kIt], own = 0;
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const int d = r0 + it * kRowsAtOnce + sub;
    chosen[it] = d < want ? kept[d] : 0;
  }
  const int dw = r0 + static_cast<int>(threadIdx.x);   // threads 0 .. kBlock - 1: a weight's row
  if (threadIdx.x < kBlock && dw < want) own = kept[dw];
  const int len = min(max(p.lens[b], 0), p.cache_len);
  const int end = min(len, p.budget);
  auto source = [&](int d, int chosen_row) {
    int s = d;
    if (len > p.budget) s = d < want ? chosen_row : len - p.budget + d;
    return min(max(s, 0), p.cache_len - 1);
  };
  if (r0 >= end) {   // uniform
    if (threadIdx.x < kBlock && dw < p.out_len) p.out_weights[pair * p.out_len + dw] = 0.f;
    return;
  }
  const int64_t stride = static_cast<int64_t>(p.hkv) * kD;
  const uint8_t* codes = p.codes[half] + (static_cast<int64_t>(b) * p.cache_len * p.hkv + h) * kD + piece * 16;
  const float* scales = p.scales[half] + pair * p.nblk;
  uint4 raw[kIt];
  float s[kIt];
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const int d = r0 + it * kRowsAtOnce + sub;
    raw[it] = make_uint4(0, 0, 0, 0);
    s[it] = 0.f;
    if (d < end) {
      const int r = source(d, chosen[it]);
      raw[it] = load_bytes<kStream, u32x4, uint4>(codes + r * stride);
      s[it] = scales[r / kBlock];
    }
  }
  float weight = 0.f;
  if (threadIdx.x < kBlock && dw < end) weight = p.weights[pair * p.cache_len + source(dw, own)];
  uint32_t amax = 0;
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    float x[16];
    decode16<kCode>(raw[it], x);
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = max(amax, abs_bits(x[j] * s[it]));
  }
  amax = half_max(amax);
  const float scale = scale_for<kCode>(amax), inv = 1.0f / scale;
  if (t == 0) p.out_scales[half][pair * p.out_nblk + jb] = scale;
  uint8_t* out = p.out_codes[half] + (static_cast<int64_t>(b) * p.out_len * p.hkv + h) * kD + piece * 16;
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const int d = r0 + it * kRowsAtOnce + sub;
    if (d < end) {
      float x[16];
      decode16<kCode>(raw[it], x);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = x[j] * s[it] * inv;
      keep_finite<kCode>(scale, x);
      *reinterpret_cast<uint4*>(out + d * stride) = encode16<kCode>(x);
    }
  }
  if (threadIdx.x < kBlock && dw < p.out_len) p.out_weights[pair * p.out_len + dw] = weight;
}

// Argument checks that the entry points share.
int check_cache(const std::string& n, int32_t batch, int64_t cache_len, int32_t heads_kv, int32_t head_dim,
                int32_t block, int32_t codes) {
  if (head_dim != kD) return invalid(n + ": head_dim must be 128");
  if (batch < 1 || cache_len < 1 || heads_kv < 1) return invalid(n + ": bad shape");
  if (batch > 65535 || heads_kv > 65535 || cache_len > INT32_MAX - 256)
    return invalid(n + ": batch, heads_kv or cache_len too large");
  if (!block_ok(block)) return invalid(n + ": block must be 16, 32, 64 or 128");
  if (codes != kE4m3 && codes != kInt8) return invalid(n + ": unknown code");
  return SWATTN_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kMaxGrid = ((int64_t{1} << 32) - 1) / 256;   // a launch has fewer than 2^32 threads

// Launch<code, block>::go(grid, stream, params...)
template <template <int, int> class Launch, class... P>
void by_code_and_block(int32_t codes, int32_t block, dim3 grid, hipStream_t st, const P&... p) {
  if (codes == kE4m3) {
    switch (block) {
      case 16: return Launch<kE4m3, 16>::go(grid, st, p...);
      case 32: return Launch<kE4m3, 32>::go(grid, st, p...);
      case 64: return Launch<kE4m3, 64>::go(grid, st, p...);
      default: return Launch<kE4m3, 128>::go(grid, st, p...);
    }
  }
  switch (block) {
    case 16: return Launch<kInt8, 16>::go(grid, st, p...);
    case 32: return Launch<kInt8, 32>::go(grid, st, p...);
    case 64: return Launch<kInt8, 64>::go(grid, st, p...);
    default: return Launch<kInt8, 128>::go(grid, st, p...);
  }
}
template <int kCode, int kBlock>
struct LaunchAppend {
  template <class Offsets>
  static void go(dim3 grid, hipStream_t st, const AppendParams& p, const Offsets& host) {
    hipLaunchKernelGGL((append_kernel<kCode, kBlock, Offsets>), grid, dim3(256), 0, st, p, host);
  }
};
template <int kCode, int kBlock>
struct LaunchGather {
  static void go(dim3 grid, hipStream_t st, const EvictParams& p, bool stream) {
    if (stream)
      hipLaunchKernelGGL((gather_kernel<kCode, kBlock, true>), grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((gather_kernel<kCode, kBlock, false>), grid, dim3(256), 0, st, p);
  }
};

}  // namespace
}  // namespace swattn

using namespace swattn;

// The checks and the launch; host: the packed offsets where they are known here, or
// null.
static int launch_append(const void* new_k, const void* new_v, const int32_t* cu_seqlens,
                        const int32_t* counts, const int32_t* cache_lens, void* k, void* v,
                        float* k_scales, float* v_scales, int32_t* lens_out, int32_t batch,
                        int64_t rows, int64_t total_rows, int64_t cache_len, int32_t heads_kv,
                        int32_t head_dim, int32_t block, int32_t codes, void* stream, const HostOffsets* host) {
  const std::string n("swattn_cache_append");
  const int st = check_cache(n, batch, cache_len, heads_kv, head_dim, block, codes);
  if (st != SWATTN_OK) return st;
  if (rows < 0 || rows > INT32_MAX || total_rows < 0 || total_rows > INT32_MAX)
    return invalid(n + ": bad number of rows");
  if (cu_seqlens != nullptr && counts != nullptr) return invalid(n + ": counts and cu_seqlens exclude each other");
  const bool any = rows > 0 && ((cu_seqlens == nullptr && host == nullptr) || total_rows > 0);
  if (cache_lens == nullptr || lens_out == nullptr || k == nullptr || v == nullptr || k_scales == nullptr ||
      v_scales == nullptr || (any && (new_k == nullptr || new_v == nullptr)))
    return invalid(n + ": null pointer");
  if (cache_lens == lens_out) return invalid(n + ": lens_out may not be cache_lens");
  if (!aligned16(k) || !aligned16(v) || (any && (!aligned16(new_k) || !aligned16(new_v))))
    return invalid(n + ": new_k, new_v, k and v must be 16-byte aligned");
  AppendParams p{};
  p.src[0] = static_cast<const uint16_t*>(new_k);
  p.src[1] = static_cast<const uint16_t*>(new_v);
  p.cu = cu_seqlens;
  p.counts = counts;
  p.lens = cache_lens;
  p.codes[0] = static_cast<uint8_t*>(k);
  p.codes[1] = static_cast<uint8_t*>(v);
  p.scales[0] = k_scales;
  p.scales[1] = v_scales;
  p.lens_out = lens_out;
  p.rows = rows;
  p.total_rows = total_rows;
  p.cache_len = static_cast<int>(cache_len);
  p.hkv = heads_kv;
  p.nblk = static_cast<int>(ceil_div(cache_len, block));
  // `rows` rows from any place of a block on; no more than the cache has.
  const int64_t most = rows < 1 ? 1 : (rows + block - 2) / block + 1;
  p.blocks = static_cast<int>(most < p.nblk ? most : p.nblk);
  const int64_t grid = static_cast<int64_t>(p.blocks) * batch * heads_kv;
  if (grid > kMaxGrid) return invalid(n + ": grid too large");
  const dim3 g(static_cast<uint32_t>(grid));
  if (host != nullptr)
    by_code_and_block<LaunchAppend>(codes, block, g, as_stream(stream), p, *host);
  else
    by_code_and_block<LaunchAppend>(codes, block, g, as_stream(stream), p, NoOffsets{});
  return launch_status(n.c_str());
}

extern "C" {

int swattn_cache_append(const void* new_k, const void* new_v, const int32_t* cu_seqlens,
                        const int32_t* counts, const int32_t* cache_lens, void* k, void* v,
                        float* k_scales, float* v_scales, int32_t* lens_out, int32_t batch,
                        int64_t rows, int64_t total_rows, int64_t cache_len, int32_t heads_kv,
                        int32_t head_dim, int32_t block, int32_t codes, void* stream) {
  return launch_append(new_k, new_v, cu_seqlens, counts, cache_lens, k, v, k_scales, v_scales, lens_out, batch,
                       rows, total_rows, cache_len, heads_kv, head_dim, block, codes, stream, nullptr);
}

int swattn_cache_append_host(const void* new_k, const void* new_v, const int32_t* cu_seqlens,
                        const int32_t* cache_lens, void* k, void* v,
                        float* k_scales, float* v_scales, int32_t* lens_out, int32_t batch,
                        int64_t rows, int64_t total_rows, int64_t cache_len, int32_t heads_kv,
                        int32_t head_dim, int32_t block, int32_t codes, void* stream) {
  if (cu_seqlens == nullptr) return invalid("swattn_cache_append: null pointer");
  if (batch < 1 || batch > SWATTN_CACHE_HOST_MAX_SEQS) return invalid("swattn_cache_append: too many sequences");
  HostOffsets host{};
  memcpy(host.cu, cu_seqlens, (static_cast<size_t>(batch) + 1) * sizeof(int32_t));
  return launch_append(new_k, new_v, nullptr, nullptr, cache_lens, k, v, k_scales, v_scales, lens_out, batch,
                       rows, total_rows, cache_len, heads_kv, head_dim, block, codes, stream, &host);
}

int swattn_cache_read(const void* k, const void* v, const float* k_scales, const float* v_scales,
                      const int32_t* starts, int64_t start, const int32_t* cache_lens, void* out_k,
                      void* out_v, int32_t batch, int64_t rows, int64_t cache_len,
                      int32_t heads_kv, int32_t head_dim, int32_t block, int32_t codes,
                      void* stream) {
  const std::string n("swattn_cache_read");
  const int st = check_cache(n, batch, cache_len, heads_kv, head_dim, block, codes);
  if (st != SWATTN_OK) return st;
  if (rows < 0 || rows > INT32_MAX || start < 0 || start > INT32_MAX) return invalid(n + ": bad range of rows");
  if (rows == 0) return SWATTN_OK;
  if (k == nullptr || v == nullptr || k_scales == nullptr || v_scales == nullptr || out_k == nullptr ||
      out_v == nullptr)
    return invalid(n + ": null pointer");
  if (!aligned16(k) || !aligned16(v) || !aligned16(out_k) || !aligned16(out_v))
    return invalid(n + ": k, v, out_k and out_v must be 16-byte aligned");
  ReadParams p{};
  p.codes[0] = static_cast<const uint8_t*>(k);
  p.codes[1] = static_cast<const uint8_t*>(v);
  p.scales[0] = k_scales;
  p.scales[1] = v_scales;
  p.starts = starts;
  p.lens = cache_lens;
  p.out[0] = static_cast<uint16_t*>(out_k);
  p.out[1] = static_cast<uint16_t*>(out_v);
  p.start = start;
  const int64_t pieces = rows * heads_kv * (kD / 16);
  if (pieces > INT32_MAX) return invalid(n + ": too many rows at once");
  p.pieces = static_cast<int32_t>(pieces);
  p.cache_len = static_cast<int>(cache_len);
  p.hkv = heads_kv;
  p.nblk = static_cast<int>(ceil_div(cache_len, block));
  p.block_log = __builtin_ctz(static_cast<unsigned>(block));
  const dim3 g(static_cast<uint32_t>(ceil_div(pieces, 256)), batch, 2);
  const bool streamed = batch * pieces * 16 * 6 >= kStreamBytes;   // K and V, codes and bf16
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, dim3(256), 0, as_stream(stream), p); };
  if (codes == kE4m3)
    streamed ? launch(read_kernel<kE4m3, true>) : launch(read_kernel<kE4m3, false>);
  else
    streamed ? launch(read_kernel<kInt8, true>) : launch(read_kernel<kInt8, false>);
  return launch_status(n.c_str());
}

size_t swattn_cache_evict_workspace_bytes(int32_t batch, int32_t heads_kv, int64_t budget) {
  if (batch < 1 || heads_kv < 1 || budget < 1) return 0;
  return (static_cast<size_t>(batch) * heads_kv * budget * sizeof(int32_t) + 255) & ~size_t{255};
}

int swattn_cache_evict(const void* k, const void* v, const float* k_scales, const float* v_scales,
                       const float* key_weights, const int32_t* cache_lens, void* out_k,
                       void* out_v, float* out_k_scales, float* out_v_scales, float* out_weights,
                       int32_t* lens_out, int32_t batch, int64_t cache_len, int64_t out_len,
                       int32_t heads_kv, int32_t head_dim, int32_t block, int32_t codes,
                       int64_t budget, int64_t recent, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const std::string n("swattn_cache_evict");
  int st = check_cache(n, batch, cache_len, heads_kv, head_dim, block, codes);
  if (st != SWATTN_OK) return st;
  st = check_cache(n, batch, out_len, heads_kv, head_dim, block, codes);
  if (st != SWATTN_OK) return st;
  if (budget < 1 || budget > out_len) return invalid(n + ": budget must lie in [1, out_len]");
  if (recent < 0 || recent > budget) return invalid(n + ": recent must lie in [0, budget]");
  if (k == nullptr || v == nullptr || k_scales == nullptr || v_scales == nullptr || key_weights == nullptr ||
      cache_lens == nullptr || out_k == nullptr || out_v == nullptr || out_k_scales == nullptr ||
      out_v_scales == nullptr || out_weights == nullptr || lens_out == nullptr)
    return invalid(n + ": null pointer");
  if (k == out_k || v == out_v || k_scales == out_k_scales || v_scales == out_v_scales ||
      key_weights == out_weights || cache_lens == lens_out)
    return invalid(n + ": the destination may not be the source");
  if (!aligned16(k) || !aligned16(v) || !aligned16(out_k) || !aligned16(out_v))
    return invalid(n + ": k, v, out_k and out_v must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < swattn_cache_evict_workspace_bytes(batch, heads_kv, budget)) {
    set_error(n + ": workspace smaller than swattn_cache_evict_workspace_bytes()");
    return SWATTN_EWORKSPACE;
  }
  if (!aligned256(workspace)) return invalid(n + ": workspace must be 256-byte aligned");
  EvictParams p{};
  p.codes[0] = static_cast<const uint8_t*>(k);
  p.codes[1] = static_cast<const uint8_t*>(v);
  p.scales[0] = k_scales;
  p.scales[1] = v_scales;
  p.weights = key_weights;
  p.lens = cache_lens;
  p.out_codes[0] = static_cast<uint8_t*>(out_k);
  p.out_codes[1] = static_cast<uint8_t*>(out_v);
  p.out_scales[0] = out_k_scales;
  p.out_scales[1] = out_v_scales;
  p.out_weights = out_weights;
  p.lens_out = lens_out;
  p.kept = static_cast<int32_t*>(workspace);
  p.cache_len = static_cast<int>(cache_len);
  p.out_len = static_cast<int>(out_len);
  p.hkv = heads_kv;
  p.nblk = static_cast<int>(ceil_div(cache_len, block));
  p.out_nblk = static_cast<int>(ceil_div(out_len, block));
  p.budget = static_cast<int>(budget);
  p.recent = static_cast<int>(recent);
  const int64_t pairs = static_cast<int64_t>(batch) * heads_kv, grid = pairs * p.out_nblk;
  if (grid > kMaxGrid || pairs > kMaxGrid / (kSelectThreads / 256)) return invalid(n + ": grid too large");
  const dim3 gs(static_cast<uint32_t>(pairs));
  const hipStream_t hs = as_stream(stream);
  // The fewest weights per thread that hold a cache, its registers and steps with them:
  // 4096 rows 5.1 us, 4097 7.2 and 5000 7.0; 8192 7.8, 16384 9.7, 16385 11.0; 32768 14.7, and
  // 32769, read again in every pass, 40 (8 pairs; 256 of 4096 rows 5.7).
  if (cache_len <= 4096)
    hipLaunchKernelGGL((select_kernel<kSelectThreads, 4>), gs, dim3(kSelectThreads), 0, hs, p);
  else if (cache_len <= 16384)
    hipLaunchKernelGGL((select_kernel<kSelectThreads, 16>), gs, dim3(kSelectThreads), 0, hs, p);
  else if (cache_len <= 32768)
    hipLaunchKernelGGL((select_kernel<kSelectThreads, 32>), gs, dim3(kSelectThreads), 0, hs, p);
  else
    hipLaunchKernelGGL((select_kernel<kSelectThreads, 0>), gs, dim3(kSelectThreads), 0, hs, p);
  // K and V, read and written.
  const bool streamed = pairs * std::min(budget, cache_len) * 4 * kD >= kStreamBytes;
  by_code_and_block<LaunchGather>(codes, block, dim3(static_cast<uint32_t>(grid)), as_stream(stream), p, streamed);
  return launch_status(n.c_str());
}

}  // extern "C"
