// The attention weight that each key received from a prefill's queries, for
// gfx950 (include/swattn_cache.h): with the forward's LSE,
//   w[b, h, j] = sum over rows i that see j, heads of the group, of
//                2^(c q_i.k_j - LSE_i).
// No counterpart in the reference, whose forward (V:103-249) leaves the log2 LSE
// (V:236-241) but not the weights.
//
// One product of the forward's two and no rescaling, with the keys stationary:
// a workgroup of four waves holds 256 keys of a KV head as MFMA A operands in
// registers, 64 per wave, and streams the 32-row blocks that can see them
// through LDS (row_blocks.h).  S^T [32 keys x 32 rows] = K Q^T by
// v_mfma_f32_32x32x16_bf16 puts a row's LSE and bounds into its own lane
// (column) and a key's sum into a register: a multiply-add, an exponential and
// an addition per pair, and the sum over lanes only once, at the end.
//
// Bound by the matrix cores and the vector ALUs together: per 32 rows and 64 keys
// a wave has 512 cycles of MFMA and about 560 of vector instructions (8 each for
// the 32 exponentials), which overlap between the two waves of a SIMD and between
// one product and the sums of the one before.  Where every row sees every key
// (S8192 Hq32/Hkv8) it runs at 1030 TFLOP/s of its 2 D flops per pair; with the
// loads and barriers taken out at 1150, the products alone at 1400, a large matrix
// product's rate.  S16384 Hq32/Hkv8 W1024 p_full 0.25: 450 us, 832 TFLOP/s; what
// lies between are blocks that a wave's keys see in part (a seventh of the local
// ones) or not at all, and the workgroups' starts.  One block per barrier, fetched
// one ahead, took 570 us; two ahead 495; the final sum by lane moves instead of
// shuffles through LDS 477; no workgroups without work 463.
//
// Rows may be cut: each list's blocks at multiples of its chunk, and a workgroup
// takes the blocks of one chunk that its keys are seen by, so that workgroups of
// different keys read the same rows at the same time.  Each leaves 256 fp32 sums,
// added in the chunks' order, the full list's first, by a last kernel: no atomics.

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <string>

#include "row_blocks.h"
#include "swattn_cache.h"
#include "swattn_internal.h"
#include "tiles.h"

namespace swattn {
namespace {

using namespace tiles;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kWaveKeys = 64;                    // two 32-key MFMA tiles
constexpr int kKeys = kWaves * kWaveKeys;        // per workgroup
constexpr int kRows = 32;                        // per block
constexpr int kBlockBytes = kRows * kRowBytes;   // 8 KiB of Q in LDS
// Row info, per block: 32 LSEs, 32 first keys, 32 key ends, 32 rows of Q (pos * hq
// + head), and the block's {largest first key, smallest end, smallest first key,
// largest end}.  A row that contributes nothing has no keys and forces the mask
// on its block.
constexpr int kInfoBytes = 576;
constexpr int kInfoLse = 0, kInfoStart = 32, kInfoEnd = 64, kInfoRow = 96, kInfoAll = 128;   // words
constexpr int kInfoLanes = (kInfoAll * 4 + 16) / 16;   // 16-byte pieces that are read
// LDS rings, in pairs of blocks: Q is fetched two pairs ahead, info three.
constexpr int kQSlots = 3, kInfoSlots = 4;
constexpr int kPairBytes = 2 * kBlockBytes, kInfoPairBytes = 2 * 1024;
constexpr int kWaitButFour = kWaitVmcnt0 | 4;   // s_waitcnt vmcnt(4)

struct WeightParams {
  const uint16_t* q;
  const uint16_t* k;
  const float* lse;
  float* out;                // [batch][hkv][seq_kv]
  const int32_t* idx[2];     // [0] full list, [1] local list
  const int32_t* starts[2];  // metadata starts per list (kMeta only)
  const int32_t* ends;       // metadata ends (kMeta only)
  int32_t count[2];          // slots per list
  int32_t nrows[2];          // count * group
  int32_t blocks[2];
  char* info;                // [hkv][blocks[0] + blocks[1]] kInfoBytes
  int32_t* ranges;           // [2][tiles][2]: the blocks of each list that see a key tile
  float* part;               // [tile][hkv][chunks][256]
  int32_t* host;             // pinned words that the lists' check reports to, one per workgroup, or null
  int32_t chunk[2], chunks[2];   // blocks per chunk and chunks of each list
  int32_t tiles, prep_wgs, check_wgs;
  int32_t seq_q, seq_kv, total_q, total_kv;
  int32_t hq, hkv, group, window;
  float c;                   // sm_scale * log2(e)
};

__device__ __forceinline__ char* block_info(const WeightParams& p, int kvh, int blk) {
  return p.info + (static_cast<int64_t>(kvh) * (p.blocks[0] + p.blocks[1]) + blk) * kInfoBytes;
}

// Row info of eight blocks of one KV head: a thread per row.
template <bool kMeta>
__device__ __forceinline__ void prep_rows(const WeightParams& p, int wg) {
  const int nblk = p.blocks[0] + p.blocks[1];
  const int per_head = (nblk + 7) >> 3;
  const int kvh = wg / per_head;
  const int blk = (wg - kvh * per_head) * 8 + (threadIdx.x >> 5);
  const int rr = threadIdx.x & 31;
  const bool in = blk < nblk;
  const int b = blk < p.blocks[0] ? 0 : 1;
  const int r = (blk - (b ? p.blocks[0] : 0)) * kRows + rr;
  bool live = in && r < p.nrows[b];
  int pos = 0, head = 0, ks = 0, ke = 0;
  if (live) {
    const int slot = r / p.group;
    head = kvh * p.group + (r - slot * p.group);
    pos = p.idx[b][slot];
    live = pos_ok(p, pos);
    if (live) row_bounds<kMeta>(p, b, pos, ks, ke);
    live = live && ks < ke;
  }
  const int64_t row = static_cast<int64_t>(pos) * p.hq + head;
  // A row that contributes nothing forces the mask on its block and widens no range.
  int max_start = live ? ks : INT_MAX, min_end = live ? ke : INT_MIN;
  int min_start = live ? ks : INT_MAX, max_end = live ? ke : INT_MIN;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    max_start = max(max_start, __shfl_xor(max_start, off));
    min_end = min(min_end, __shfl_xor(min_end, off));
    min_start = min(min_start, __shfl_xor(min_start, off));
    max_end = max(max_end, __shfl_xor(max_end, off));
  }
  if (!in) return;
  char* inf = block_info(p, kvh, blk);
  float* words = reinterpret_cast<float*>(inf);
  int* ints = reinterpret_cast<int*>(inf);
  words[kInfoLse + rr] = live ? p.lse[row] : 0.f;
  ints[kInfoStart + rr] = live ? ks : 0;
  ints[kInfoEnd + rr] = live ? ke : 0;
  ints[kInfoRow + rr] = live ? static_cast<int>(row) : 0;
  if (rr == 0) *reinterpret_cast<int4*>(ints + kInfoAll) = make_int4(max_start, min_end, min_start, max_end);
}

// The check of the lists, reported to a host that polls: the word carries the
// answer itself and orders nothing else.  As many rows are listed as there are, so that
// disjoint lists hold every row: entry i of the full list, row x, has x - i rows of the
// local list before it.  Two loads in place of a search: S1024 18.6 -> 17.9 us.  (In the
// next launch, where it would delay no kernel: 26.1, the host's answer comes late.)
constexpr int kReported = 1 << 30;
__device__ __forceinline__ void check_lists(const WeightParams& p, int wg) {
  int f = 0;
  const int64_t nf = p.count[0], nl = p.count[1];
  const int32_t *full = p.idx[0], *local = p.idx[1];
  for (int64_t i = static_cast<int64_t>(wg) * kThreads + threadIdx.x; i < max(nf, nl);
       i += static_cast<int64_t>(p.check_wgs) * kThreads) {
    if (i < nf) {
      const int64_t x = full[i], before = x - i;   // of the local list
      if (x < 0 || x >= p.total_q) f |= SWATTN_ERR_FULL_RANGE;
      if (i > 0 && x <= full[i - 1]) f |= SWATTN_ERR_FULL_ORDER;
      if (before < 0 || before > nl || (before > 0 && local[before - 1] >= x) || (before < nl && local[before] <= x))
        f |= SWATTN_ERR_OVERLAP;
    }
    if (i < nl) {
      const int32_t x = local[i];
      if (x < 0 || x >= p.total_q) f |= SWATTN_ERR_LOCAL_RANGE;
      if (i > 0 && x <= local[i - 1]) f |= SWATTN_ERR_LOCAL_ORDER;
    }
  }
  __shared__ int s_flags[kThreads / 64];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) f |= __shfl_xor(f, off);
  if ((threadIdx.x & 63) == 0) s_flags[threadIdx.x >> 6] = f;
  __syncthreads();
  if (threadIdx.x == 0)
    __hip_atomic_store(p.host + wg, s_flags[0] | s_flags[1] | s_flags[2] | s_flags[3] | kReported,
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// The lists' check, row info and block ranges need nothing of each other: one
// launch.
template <bool kMeta>
__global__ __launch_bounds__(kThreads) void weights_prep_kernel(const WeightParams p) {
  const int wg = static_cast<int>(blockIdx.x) - p.check_wgs;
  if (wg < 0)
    check_lists(p, blockIdx.x);
  else if (wg < p.prep_wgs)
    prep_rows<kMeta>(p, wg);
  else
    block_ranges<kMeta, kKeys, kRows>(p, p.tiles, wg - p.prep_wgs);
}

// The x-th workgroup of key tile t: the list and chunk that it takes and the blocks
// of that chunk that see the tile, [a, a_end) on the axis of both lists.  Chunks of
// the full list come first, from its end on, which every tile shares.
struct Share {
  int part, a, a_end;
};
__device__ __forceinline__ bool chunk_share(const WeightParams& p, int t, int x, Share& sh) {
  const int2 f = *reinterpret_cast<const int2*>(p.ranges + 2 * t);
  const int2 l = *reinterpret_cast<const int2*>(p.ranges + 2 * (p.tiles + t));
  const int f_last = f.x < f.y ? (f.y - 1) / p.chunk[0] : -1, f_first = f.x < f.y ? f.x / p.chunk[0] : 0;
  const int nf = f_last - f_first + 1;
  const int b = x < nf ? 0 : 1;
  if (b == 1 && l.x >= l.y) return false;
  const int c = b == 0 ? f_last - x : l.x / p.chunk[1] + (x - nf);
  const int2 r = b == 0 ? f : l;
  const int lo = c * p.chunk[b], hi = lo + p.chunk[b];
  if (lo >= r.y) return false;
  sh.part = b == 0 ? c : p.chunks[0] + c;
  const int base = b == 0 ? 0 : p.blocks[0];
  sh.a = base + max(r.x, lo);
  sh.a_end = base + min(r.y, hi);
  return true;
}

// One workgroup per (share, key tile, KV head), KV head fastest.
__global__ __launch_bounds__(kThreads, 2) void weights_kernel(const WeightParams p) {
  __shared__ __align__(16) char smem[kQSlots * kPairBytes + kInfoSlots * kInfoPairBytes];
  const int kvh = blockIdx.x % p.hkv;
  const int rest = blockIdx.x / p.hkv;
  const int t = rest % p.tiles;
  Share sh;
  if (!chunk_share(p, t, rest / p.tiles, sh)) return;   // uniform
  const int n = sh.a_end - sh.a;   // at least 1
  auto block_at = [&](int i) { return sh.a + i; };
  const int tid = threadIdx.x, lane = tid & 63;
  auto uniform = [](uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); };
  const int wave = static_cast<int>(uniform(tid >> 6));
  const int r = lane & 31, hh = lane >> 5;
  const int key0 = t * kKeys + wave * kWaveKeys;
  // K operands: key r of each 32-key tile, dims 16 x + 8 hh .. +7.
  bf16x8 kf[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t key = min(key0 + 32 * u + r, p.total_kv - 1);
    const uint16_t* row = p.k + (key * p.hkv + kvh) * kD + 8 * hh;
#pragma unroll
    for (int x = 0; x < 8; ++x) kf[u][x] = *reinterpret_cast<const bf16x8*>(row + 16 * x);
  }
  // Staging.  Waves 0 and 1 fetch the info of a pair's blocks; every wave 16 of its
  // 64 rows, four per 1 KiB load: LDS chunk position lane % 16 of row rr takes the
  // row's chunk (lane % 16) ^ swz(rr).
  char* const s_info = smem + kQSlots * kPairBytes;
  auto stage_info = [&](int i) {
    if (wave < 2 && lane < kInfoLanes)
      dma16_gather(block_info(p, kvh, block_at(min(2 * i + wave, n - 1))) + 16 * lane,
                   uniform(lds_addr(s_info) + (i % kInfoSlots) * kInfoPairBytes + wave * 1024));
  };
  const int stage_row = 16 * (wave & 1) + (lane >> 4);   // of block wave / 2
  auto stage_rows = [&](int i) {
    const int* rows = reinterpret_cast<const int*>(s_info + (i % kInfoSlots) * kInfoPairBytes + (wave >> 1) * 1024) + kInfoRow;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int rr = stage_row + 4 * x;
      const uint16_t* src = p.q + static_cast<int64_t>(rows[rr]) * kD + 8 * ((lane & 15) ^ swz(rr));
      dma16_gather(src, uniform(lds_addr(smem) + (i % kQSlots) * kPairBytes + wave * 4096 + 1024 * x));
    }
  };
  stage_info(0);
  stage_info(1);
  stage_info(2);
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
  __syncthreads();
  stage_rows(0);
  stage_rows(1);
  f32x16 sum[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[u][x] = 0.f;
  auto product = [&](int u, const bf16x8 (&q)[8], f32x16& d) {
#pragma unroll
    for (int x = 0; x < 16; ++x) d[x] = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u][x], q[x], d, 0, 0, 0);
  };
  auto add = [&](int u, float row_lse, const f32x16& d) {
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[u][x] += __builtin_amdgcn_exp2f(__builtin_fmaf(d[x], p.c, -row_lse));
  };
  // The last product of a pair is summed up beside the next pair's first: d1, of
  // rows with LSE lse_p (infinite: nothing left to sum).
  f32x16 d0, d1;
  float lse_p = INFINITY;
#pragma unroll
  for (int x = 0; x < 16; ++x) d1[x] = 0.f;
  const int pairs = (n + 1) >> 1;
  for (int i = 0; i < pairs; ++i) {
    // All but this wave's last four loads (rows of pair i + 1) are there: its rows
    // of pair i and its info of pair i + 2; after the barrier, everyone's.  Pair
    // i - 1's rows and info, whose slots are filled next, were last read before it.
    __builtin_amdgcn_s_waitcnt(kWaitButFour);
    __syncthreads();
    stage_info(i + 3);
    const char* inf = s_info + (i % kInfoSlots) * kInfoPairBytes;
    int4 all[2];
    float lse[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      all[y] = *reinterpret_cast<const int4*>(inf + 1024 * y + 4 * kInfoAll);
      lse[y] = reinterpret_cast<const float*>(inf + 1024 * y)[kInfoLse + r];
    }
    bool none[2], whole[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int max_start = __builtin_amdgcn_readfirstlane(all[y].x), min_end = __builtin_amdgcn_readfirstlane(all[y].y);
      const int min_start = __builtin_amdgcn_readfirstlane(all[y].z), max_end = __builtin_amdgcn_readfirstlane(all[y].w);
      none[y] = max_end <= key0 || min_start >= key0 + kWaveKeys || 2 * i + y >= n;
      whole[y] = max_start <= key0 && min_end >= key0 + kWaveKeys && 2 * i + y < n;
    }
    const char* slot = smem + (i % kQSlots) * kPairBytes + r * kRowBytes;
    auto q_at = [&](int y, int x) { return *reinterpret_cast<const bf16x8*>(slot + y * kBlockBytes + 16 * ((2 * x + hh) ^ swz(r))); };
    bf16x8 qf[8];
    if (whole[0] && whole[1]) {   // every row sees every key
#pragma unroll
      for (int x = 0; x < 8; ++x) qf[x] = q_at(0, x);
      stage_rows(i + 2);
      product(0, qf, d0);
      add(1, lse_p, d1);
      product(1, qf, d1);
      add(0, lse[0], d0);
#pragma unroll
      for (int x = 0; x < 8; ++x) qf[x] = q_at(1, x);
      product(0, qf, d0);
      add(1, lse[0], d1);
      product(1, qf, d1);
      add(0, lse[1], d0);
      lse_p = lse[1];
      continue;
    }
    stage_rows(i + 2);
    add(1, lse_p, d1);   // what the last pair left
    lse_p = INFINITY;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      if (none[y]) continue;
#pragma unroll
      for (int x = 0; x < 8; ++x) qf[x] = q_at(y, x);
      if (whole[y]) {
        product(0, qf, d0);
        product(1, qf, d1);
        add(0, lse[y], d0);
        add(1, lse[y], d1);
        continue;
      }
      const int ks = reinterpret_cast<const int*>(inf + 1024 * y)[kInfoStart + r];
      const int ke = reinterpret_cast<const int*>(inf + 1024 * y)[kInfoEnd + r];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        product(u, qf, d0);
        const int first = ks - key0 - 32 * u - 4 * hh;
        const uint32_t keys = ke - ks;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(d0[x], p.c, -lse[y]));
          sum[u][x] += static_cast<uint32_t>(8 * (x >> 2) + (x & 3) - first) < keys ? w : 0.f;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) d1[x] = 0.f;
  }
  add(1, lse_p, d1);
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);   // no load into LDS outlives the workgroup
  // Sums over the 32 row lanes, with lane moves only: neighbours, pairs, the mirror
  // image within 8 and 16 lanes, and the other 16.
  float* out = p.part + ((static_cast<int64_t>(t) * p.hkv + kvh) * (p.chunks[0] + p.chunks[1]) + sh.part) * kKeys + wave * kWaveKeys;
  float mine = 0.f;   // lane r: element r % 16 of tile r / 16
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      constexpr int kMoves[4] = {0xB1, 0x4E, 0x141, 0x140};
      float w = sum[u][x];
      w += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w), kMoves[0], 0xf, 0xf, false));
      w += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w), kMoves[1], 0xf, 0xf, false));
      w += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w), kMoves[2], 0xf, 0xf, false));
      w += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w), kMoves[3], 0xf, 0xf, false));
      const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(w), __float_as_uint(w), false, false);
      w = __uint_as_float(both[0]) + __uint_as_float(both[1]);
      mine = r == 16 * u + x ? w : mine;
    }
  out[32 * (r >> 4) + 8 * ((r & 15) >> 2) + 4 * hh + (r & 3)] = mine;
}

// The chunks' sums, in their order: one workgroup per (key tile, KV head), a thread
// per key.
__global__ __launch_bounds__(kThreads) void weights_reduce_kernel(const WeightParams p) {
  const int kvh = blockIdx.x % p.hkv, t = blockIdx.x / p.hkv;
  const int key = t * kKeys + threadIdx.x;
  const float* part = p.part + (static_cast<int64_t>(t) * p.hkv + kvh) * (p.chunks[0] + p.chunks[1]) * kKeys + threadIdx.x;
  float w = 0.f;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int2 r = *reinterpret_cast<const int2*>(p.ranges + 2 * (b * p.tiles + t));
    if (r.x >= r.y) continue;
    const int end = (r.y - 1) / p.chunk[b] + 1;
    for (int s = r.x / p.chunk[b]; s < end; ++s) w += part[static_cast<int64_t>(b * p.chunks[0] + s) * kKeys];
  }
  if (key < p.total_kv) {
    const int b = key / p.seq_kv;
    p.out[(static_cast<int64_t>(b) * p.hkv + kvh) * p.seq_kv + (key - b * p.seq_kv)] = w;
  }
}

struct Layout {
  int64_t tiles, blocks[2], chunk[2], chunks[2];
  size_t off_ranges, off_part, bytes;
};

// Chunks: on small grids about as many workgroups with work as run at once (two per
// CU; half of the chunks see nothing), one block longer since a pair's first and last
// chunks are partial; on large grids short enough that the workgroups outnumber the
// slots several times over, the local list's half as long, since they run last.
// Workgroups wanted in all, 768, 1024 and 1024 with the block more: S2048 Hq32/Hkv8
// 39.4 us, 36.8, 35.9; S3333 Hq24/Hkv3 71.5, -, 62.7; B4 S1024 Hq16/Hkv8 39.0, 36.4,
// 38.8; B2 S980 Hq8/Hkv2 22.8, 26.8, 22.4; 640 and 1280 are slower nearly everywhere.
// (S16384, full and local chunks of 128 and 64 460 us, 64 and 64 466, 64 and 32 467,
// 128 and 32 462; one long line of blocks cut into equal shares, 2 to 8 per CU, 479 to
// 467, and S1024 19.6 instead of 17.0.)
constexpr int64_t kMinChunk = 4;
constexpr int64_t kMaxChunk = 128;
constexpr int64_t kWantWgs = 1024;
constexpr int64_t kMaxPartBytes = int64_t{64} << 20;

Layout layout(int64_t total_kv, int64_t heads_kv, int64_t group, int64_t n_full, int64_t n_local) {
  Layout L{};
  L.tiles = ceil_div(total_kv, kKeys);
  L.blocks[0] = ceil_div(n_full * group, kRows);
  L.blocks[1] = ceil_div(n_local * group, kRows);
  const int64_t axis = std::max<int64_t>(1, L.blocks[0] + L.blocks[1]);
  const int64_t pairs = L.tiles * heads_kv;
  int64_t chunk = std::min(kMaxChunk, std::max(kMinChunk, ceil_div(axis * pairs, kWantWgs) + 1));
  const int64_t most = std::max<int64_t>(2, kMaxPartBytes / (pairs * kKeys * 4));   // chunks per pair
  chunk = std::max(chunk, ceil_div(3 * axis, 2 * most));
  L.chunk[0] = chunk;
  L.chunk[1] = chunk >= 64 ? chunk / 2 : chunk;
  for (int b = 0; b < 2; ++b) L.chunks[b] = ceil_div(L.blocks[b], L.chunk[b]);
  auto al = [](size_t x) { return (x + 255) & ~size_t{255}; };
  size_t o = al(static_cast<size_t>(axis * heads_kv) * kInfoBytes);
  L.off_ranges = o;  o = al(o + static_cast<size_t>(2 * L.tiles) * 2 * sizeof(int32_t));
  L.off_part = o;    o = al(o + static_cast<size_t>(pairs * (L.chunks[0] + L.chunks[1])) * kKeys * sizeof(float));
  L.bytes = o;
  return L;
}

// Workgroups that check the lists, each with a word to report to.
int check_wgs(int64_t slots) {
  return static_cast<int>(std::min<int64_t>(SWATTN_KEY_WEIGHTS_HOST_WORDS, ceil_div(slots, kThreads)));
}

}  // namespace
}  // namespace swattn

using namespace swattn;
using namespace swattn::tiles;

// The checks and the launches; host: pinned words for the lists' check, or null.
static int launch_key_weights(
    const void* q, const void* k, const float* lse, const int32_t* full_idx, int64_t n_full,
    const int32_t* local_idx, int64_t n_local, const int32_t* full_starts, const int32_t* local_starts,
    const int32_t* causal_ends, float* key_weights, int32_t batch, int64_t seq_q, int64_t seq_kv,
    int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t window, float scale_log2, void* workspace,
    size_t workspace_bytes, void* stream, int32_t* host) {
  const std::string n("swattn_prefill_key_weights");
  if (head_dim != kD) return invalid(n + ": head_dim must be 128");
  if (batch < 1 || seq_q < 0 || seq_kv < 1 || heads_q < 1 || heads_kv < 1) return invalid(n + ": bad shape");
  if (heads_q % heads_kv != 0) return invalid(n + ": heads_q must be a multiple of heads_kv");
  if (heads_kv > 4096 || heads_q > 65536) return invalid(n + ": at most 4096 KV heads and 65536 query heads");
  if (window <= 0) return invalid(n + ": window must be positive");
  if (!isfinite(scale_log2)) return invalid(n + ": scale_log2 must be finite");
  if (seq_q > INT32_MAX || seq_kv > INT32_MAX) return invalid(n + ": batch*seq must stay below 2^31");
  const int64_t total_q = static_cast<int64_t>(batch) * seq_q, total_kv = static_cast<int64_t>(batch) * seq_kv;
  if (total_q > INT32_MAX || total_kv > INT32_MAX - 2 * kKeys) return invalid(n + ": batch*seq must stay below 2^31");
  if (n_full < 0 || n_local < 0 || n_full > total_q || n_local > total_q - n_full)
    return invalid(n + ": bad index counts");
  const int64_t group = heads_q / heads_kv;
  if ((n_full + n_local) * group > INT32_MAX - 2 * kRows) return invalid(n + ": too many rows");
  if (total_q * heads_q > INT32_MAX) return invalid(n + ": more than 2^31 - 1 rows of Q");
  const bool meta = full_starts != nullptr || local_starts != nullptr || causal_ends != nullptr;
  if (meta && (full_starts == nullptr || local_starts == nullptr || causal_ends == nullptr))
    return invalid(n + ": metadata needs full_starts, local_starts and causal_ends");
  if (k == nullptr || key_weights == nullptr ||
      (n_full + n_local > 0 && (q == nullptr || lse == nullptr || (n_full > 0 && full_idx == nullptr) ||
                                (n_local > 0 && local_idx == nullptr))))
    return invalid(n + ": null pointer");
  if (!aligned16(k) || (n_full + n_local > 0 && !aligned16(q))) return invalid(n + ": q and k must be 16-byte aligned");
  const Layout L = layout(total_kv, heads_kv, group, n_full, n_local);
  if (workspace == nullptr || workspace_bytes < L.bytes) {
    set_error(n + ": workspace smaller than swattn_prefill_key_weights_workspace_bytes()");
    return SWATTN_EWORKSPACE;
  }
  if (!aligned256(workspace)) return invalid(n + ": workspace must be 256-byte aligned");
  // Workgroups per tile: chunks of the full list, and of the local rows between the
  // first and the last that see the tile: for each sequence in it window - 1 positions
  // more than its keys there, or those behind the sequence's last key, which may see none.
  int64_t local = L.blocks[1];
  if (!meta) {
    const int64_t reach = std::min(std::max<int64_t>(window, seq_q - seq_kv), seq_q), parts = kKeys / seq_kv + 2;
    local = std::min(local, (kKeys + parts * reach) * group / kRows + 2);
  }
  const int64_t shares = L.chunks[0] + std::min(L.chunks[1], ceil_div(local, L.chunk[1]) + 1);
  const int64_t pairs = L.tiles * heads_kv, grid = pairs * std::max<int64_t>(shares, 1);
  const int64_t prep = ceil_div(L.blocks[0] + L.blocks[1], 8) * heads_kv, ranges = ceil_div(2 * L.tiles, kThreads / 64);
  constexpr int64_t kMaxGrid = ((int64_t{1} << 32) - 1) / kThreads;   // a launch has fewer than 2^32 threads
  if (grid > kMaxGrid || prep + ranges > kMaxGrid - SWATTN_KEY_WEIGHTS_HOST_WORDS) return invalid(n + ": grid too large");
  char* ws = static_cast<char*>(workspace);
  WeightParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.lse = lse;
  p.out = key_weights;
  p.idx[0] = full_idx;
  p.idx[1] = local_idx;
  p.starts[0] = full_starts;
  p.starts[1] = local_starts;
  p.ends = causal_ends;
  p.count[0] = static_cast<int32_t>(n_full);
  p.count[1] = static_cast<int32_t>(n_local);
  for (int b = 0; b < 2; ++b) {
    p.nrows[b] = static_cast<int32_t>(p.count[b] * group);
    p.blocks[b] = static_cast<int32_t>(L.blocks[b]);
  }
  p.info = ws;
  p.ranges = reinterpret_cast<int32_t*>(ws + L.off_ranges);
  p.part = reinterpret_cast<float*>(ws + L.off_part);
  p.tiles = static_cast<int32_t>(L.tiles);
  for (int b = 0; b < 2; ++b) {
    p.chunk[b] = static_cast<int32_t>(L.chunk[b]);
    p.chunks[b] = static_cast<int32_t>(L.chunks[b]);
  }
  p.prep_wgs = static_cast<int32_t>(prep);
  p.seq_q = static_cast<int32_t>(seq_q);
  p.seq_kv = static_cast<int32_t>(seq_kv);
  p.total_q = static_cast<int32_t>(total_q);
  p.total_kv = static_cast<int32_t>(total_kv);
  p.hq = heads_q;
  p.hkv = heads_kv;
  p.group = static_cast<int32_t>(group);
  p.window = window;
  p.c = scale_log2;
  const hipStream_t st = as_stream(stream);
  p.host = host;
  p.check_wgs = host == nullptr ? 0 : check_wgs(std::max(n_full, n_local));
  const dim3 gp(static_cast<uint32_t>(p.check_wgs + prep + ranges));
  if (meta)
    hipLaunchKernelGGL(weights_prep_kernel<true>, gp, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL(weights_prep_kernel<false>, gp, dim3(kThreads), 0, st, p);
  hipLaunchKernelGGL(weights_kernel, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), 0, st, p);
  hipLaunchKernelGGL(weights_reduce_kernel, dim3(static_cast<uint32_t>(pairs)), dim3(kThreads), 0, st, p);
  return launch_status(n.c_str());
}

extern "C" {

size_t swattn_prefill_key_weights_workspace_bytes(int32_t batch, int64_t seq_kv, int32_t heads_q,
                                                  int32_t heads_kv, int32_t head_dim, int64_t n_full,
                                                  int64_t n_local) {
  if (batch < 1 || seq_kv < 1 || seq_kv > INT32_MAX || heads_q < 1 || heads_kv < 1 || heads_q % heads_kv ||
      head_dim != kD || n_full < 0 || n_local < 0 || n_full > INT32_MAX || n_local > INT32_MAX)
    return 0;
  return layout(batch * seq_kv, heads_kv, heads_q / heads_kv, n_full, n_local).bytes;
}

int swattn_prefill_key_weights(
    const void* q, const void* k, const float* lse, const int32_t* full_idx, int64_t n_full,
    const int32_t* local_idx, int64_t n_local, const int32_t* full_starts, const int32_t* local_starts,
    const int32_t* causal_ends, float* key_weights, int32_t batch, int64_t seq_q, int64_t seq_kv,
    int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t window, float scale_log2, void* workspace,
    size_t workspace_bytes, void* stream) {
  return launch_key_weights(q, k, lse, full_idx, n_full, local_idx, n_local, full_starts, local_starts, causal_ends,
                     key_weights, batch, seq_q, seq_kv, heads_q, heads_kv, head_dim, window, scale_log2,
                     workspace, workspace_bytes, stream, nullptr);
}

int swattn_prefill_key_weights_checked(
    const void* q, const void* k, const float* lse, const int32_t* full_idx, int64_t n_full,
    const int32_t* local_idx, int64_t n_local, const int32_t* full_starts, const int32_t* local_starts,
    const int32_t* causal_ends, float* key_weights, int32_t batch, int64_t seq_q, int64_t seq_kv,
    int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t window, float scale_log2, void* workspace,
    size_t workspace_bytes, void* stream, int32_t* host, int32_t* flags) {
  const std::string n("swattn_prefill_key_weights");
  if (host == nullptr || flags == nullptr) return invalid(n + ": null pointer");
  *flags = 0;
  if (n_full + n_local != batch * seq_q) return invalid(n + ": the lists must hold batch * seq_q entries");
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(as_stream(stream), &capture) == hipSuccess && capture != hipStreamCaptureStatusNone)
    return invalid(n + ": waits for the check of the index lists and cannot be captured");
  const int words = n_full < 0 || n_local < 0 ? 0 : check_wgs(std::max(n_full, n_local));
  for (int i = 0; i < words; ++i) host[i] = 0;
  const int status = launch_key_weights(q, k, lse, full_idx, n_full, local_idx, n_local, full_starts, local_starts,
                                 causal_ends, key_weights, batch, seq_q, seq_kv, heads_q, heads_kv, head_dim,
                                 window, scale_log2, workspace, workspace_bytes, stream, host);
  if (status != SWATTN_OK) {
    // After a HIP error a kernel may be queued all the same, and must not report
    // into the next call's words.
    if (status > 0) (void)hipStreamSynchronize(as_stream(stream));
    return status;
  }
  // Poll for a while (the stream may hold any amount of earlier work, or have
  // failed), then wait for the stream.
  volatile int32_t* word = host;
  const auto t0 = std::chrono::steady_clock::now();
  int done = 0;
  while (done < words) {
    if (word[done] != 0) {
      *flags |= word[done++] & ~kReported;
      continue;
    }
    __builtin_ia32_pause();
    if (std::chrono::steady_clock::now() - t0 > std::chrono::milliseconds(2)) break;
  }
  if (done == words) return SWATTN_OK;
  const hipError_t e = hipStreamSynchronize(as_stream(stream));
  if (e != hipSuccess) {
    set_error(n + ": " + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  for (; done < words; ++done) *flags |= word[done] & ~kReported;
  return SWATTN_OK;
}

}  // extern "C"
