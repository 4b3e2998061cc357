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
// Rows may be cut: the blocks of both lists form one axis (full first), cut at
// multiples of `chunk` blocks, and a workgroup takes the blocks of one chunk that
// its keys are seen by, so that workgroups of different keys read the same rows
// at the same time.  Each leaves 256 fp32 sums, added in the chunks' order by
// a last kernel: no atomics.

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <string>

#include "row_blocks.h"
#include "swattn_cache.h"
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
constexpr int kSlots = 2;
// Row info, per block: 32 LSEs, 32 first keys, 32 key ends, 32 element offsets in
// Q (-1: a row that contributes nothing), and the block's {largest first key,
// smallest end, smallest first key, largest end}.
constexpr int kInfoBytes = 768;
constexpr int kInfoLse = 0, kInfoStart = 32, kInfoEnd = 64, kInfoAll = 160;   // words
constexpr int kInfoOff = 48;                                                  // int64s

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
  uint16_t* zero_row;        // 128 zeros: the source of rows that contribute nothing
  int32_t* ranges;           // [2][tiles][2]: the blocks of each list that see a key tile
  float* part;               // [tile][hkv][chunks][256]
  int32_t tiles, chunk, chunks, prep_wgs;
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
  if (wg == 0 && threadIdx.x < kRowBytes / 16)
    reinterpret_cast<uint4*>(p.zero_row)[threadIdx.x] = make_uint4(0, 0, 0, 0);
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
  reinterpret_cast<int64_t*>(inf)[kInfoOff + rr] = live ? row * kD : -1;
  if (rr == 0) *reinterpret_cast<int4*>(ints + kInfoAll) = make_int4(max_start, min_end, min_start, max_end);
}

// Row info and block ranges need nothing of each other: one launch.
template <bool kMeta>
__global__ __launch_bounds__(kThreads) void weights_prep_kernel(const WeightParams p) {
  const int wg = blockIdx.x;
  if (wg < p.prep_wgs)
    prep_rows<kMeta>(p, wg);
  else
    block_ranges<kMeta, kKeys, kRows>(p, p.tiles, wg - p.prep_wgs);
}

// The blocks of chunk s, on the axis of both lists, that see tile t: [a, a_end)
// of the full list, then [b, b_end) of the local one.
struct Share {
  int a, a_end, b, b_end;
};
__device__ __forceinline__ Share chunk_share(const WeightParams& p, int t, int s) {
  const int lo = s * p.chunk, hi = lo + p.chunk;
  const int32_t* f = p.ranges + 2 * t;
  const int32_t* l = p.ranges + 2 * (p.tiles + t);
  Share x;
  x.a = max(f[0], lo);
  x.a_end = max(min(f[1], hi), x.a);
  x.b = max(l[0] + p.blocks[0], lo);
  x.b_end = max(min(l[1] + p.blocks[0], hi), x.b);
  return x;
}

// One workgroup per (chunk, key tile, KV head), KV head fastest.
__global__ __launch_bounds__(kThreads, 2) void weights_kernel(const WeightParams p) {
  __shared__ __align__(16) char smem[kSlots * kBlockBytes];
  const int kvh = blockIdx.x % p.hkv;
  const int rest = blockIdx.x / p.hkv;
  const int t = rest % p.tiles, s = rest / p.tiles;
  const Share sh = chunk_share(p, t, s);
  const int na = sh.a_end - sh.a, n = na + sh.b_end - sh.b;
  if (n <= 0) return;   // uniform
  auto block_at = [&](int i) { return i < na ? sh.a + i : sh.b + (i - na); };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
  // Staging: this wave's two 1 KiB loads of a block, four rows each; LDS chunk
  // position lane % 16 of row rr takes the row's chunk (lane % 16) ^ swz(rr).
  const int stage_row = 8 * wave + (lane >> 4);
  const uint32_t lds0 = lds_addr(smem) + wave * 2048;
  auto offsets = [&](int i, int64_t (&off)[2]) {
    const int64_t* o = reinterpret_cast<const int64_t*>(block_info(p, kvh, block_at(min(i, n - 1)))) + kInfoOff;
    off[0] = o[stage_row];
    off[1] = o[stage_row + 4];
  };
  auto stage = [&](int i, const int64_t (&off)[2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int c = (lane & 15) ^ swz(stage_row + 4 * x);
      const uint16_t* src = (off[x] >= 0 ? p.q + off[x] : p.zero_row) + 8 * c;
      dma16_gather(src, lds0 + (i % kSlots) * kBlockBytes + 1024 * x);
    }
  };
  struct RowInfo {
    float lse;
    int ks, ke;
    int4 all;
  };
  auto row_info = [&](int i) {
    const int* w = reinterpret_cast<const int*>(block_info(p, kvh, block_at(min(i, n - 1))));
    RowInfo x;
    x.lse = __int_as_float(w[kInfoLse + r]);
    x.ks = w[kInfoStart + r];
    x.ke = w[kInfoEnd + r];
    x.all = *reinterpret_cast<const int4*>(w + kInfoAll);
    return x;
  };
  int64_t off[2];
  offsets(0, off);
  stage(0, off);
  offsets(1, off);
  RowInfo next = row_info(0);
  f32x16 sum[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[u][x] = 0.f;
  for (int i = 0; i < n; ++i) {
    // This wave's part of block i is there, and after the barrier all of it; the
    // slot of block i + 1 was last read for block i - 1, before the barrier.
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    __syncthreads();
    const RowInfo info = next;
    if (i + 1 < n) {
      stage(i + 1, off);
      offsets(i + 2, off);
      next = row_info(i + 1);
    }
    const int max_start = __builtin_amdgcn_readfirstlane(info.all.x), min_end = __builtin_amdgcn_readfirstlane(info.all.y);
    const int min_start = __builtin_amdgcn_readfirstlane(info.all.z), max_end = __builtin_amdgcn_readfirstlane(info.all.w);
    if (max_end <= key0 || min_start >= key0 + kWaveKeys) continue;   // none of this wave's keys
    const char* blk = smem + (i % kSlots) * kBlockBytes + r * kRowBytes;
    bf16x8 qf[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) qf[x] = *reinterpret_cast<const bf16x8*>(blk + 16 * ((2 * x + hh) ^ swz(r)));
    f32x16 d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int x = 0; x < 16; ++x) d[u][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) d[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u][x], qf[x], d[u], 0, 0, 0);
    }
    if (max_start <= key0 && min_end >= key0 + kWaveKeys) {   // every row sees every key
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 0; x < 16; ++x) sum[u][x] += __builtin_amdgcn_exp2f(__builtin_fmaf(d[u][x], p.c, -info.lse));
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int key = key0 + 32 * u + 8 * (x >> 2) + 4 * hh + (x & 3);
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(d[u][x], p.c, -info.lse));
          sum[u][x] += key >= info.ks && key < info.ke ? w : 0.f;
        }
    }
  }
  // Sums over the 32 row lanes; lane 0 of each half holds its keys'.
  float* out = p.part + ((static_cast<int64_t>(t) * p.hkv + kvh) * p.chunks + s) * kKeys + wave * kWaveKeys;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      float w = sum[u][x];
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) w += __shfl_xor(w, o);
      if (r == 0) out[32 * u + 8 * (x >> 2) + 4 * hh + (x & 3)] = w;
    }
}

// The chunks' sums, in their order: one workgroup per (key tile, KV head), a thread
// per key.
__global__ __launch_bounds__(kThreads) void weights_reduce_kernel(const WeightParams p) {
  const int kvh = blockIdx.x % p.hkv, t = blockIdx.x / p.hkv;
  const int key = t * kKeys + threadIdx.x;
  const int32_t* f = p.ranges + 2 * t;
  const int32_t* l = p.ranges + 2 * (p.tiles + t);
  const float* part = p.part + (static_cast<int64_t>(t) * p.hkv + kvh) * p.chunks * kKeys + threadIdx.x;
  float w = 0.f;
  int from = 0;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int lo = (b ? l[0] + p.blocks[0] : f[0]), hi = (b ? l[1] + p.blocks[0] : f[1]);
    if (lo >= hi) continue;
    const int end = (hi - 1) / p.chunk + 1;
    for (int s = max(lo / p.chunk, from); s < end; ++s) w += part[static_cast<int64_t>(s) * kKeys];
    from = end;   // a chunk that holds blocks of both lists counts once
  }
  if (key < p.total_kv) {
    const int b = key / p.seq_kv;
    p.out[(static_cast<int64_t>(b) * p.hkv + kvh) * p.seq_kv + (key - b * p.seq_kv)] = w;
  }
}

struct Layout {
  int64_t tiles, blocks[2], chunk, chunks;
  size_t off_zero, off_ranges, off_part, bytes;
};

// Chunks: short enough that the workgroups outnumber the chip's slots several
// times over, long enough that the partial sums stay small.
constexpr int64_t kMinChunk = 8;
constexpr int64_t kMaxChunk = 64;
constexpr int64_t kWantWgs = 4096;                // workgroups, if all chunks had blocks
constexpr int64_t kMaxPartBytes = int64_t{64} << 20;

Layout layout(int64_t total_kv, int64_t heads_kv, int64_t group, int64_t n_full, int64_t n_local) {
  Layout L{};
  L.tiles = ceil_div(total_kv, kKeys);
  L.blocks[0] = ceil_div(n_full * group, kRows);
  L.blocks[1] = ceil_div(n_local * group, kRows);
  const int64_t axis = std::max<int64_t>(1, L.blocks[0] + L.blocks[1]);
  const int64_t pairs = L.tiles * heads_kv;
  L.chunk = std::min(kMaxChunk, std::max(kMinChunk, ceil_div(axis * pairs, kWantWgs)));
  const int64_t most = std::max<int64_t>(1, kMaxPartBytes / (pairs * kKeys * 4));   // chunks per pair
  L.chunk = std::max(L.chunk, ceil_div(axis, most));
  L.chunks = ceil_div(axis, L.chunk);
  auto al = [](size_t x) { return (x + 255) & ~size_t{255}; };
  size_t o = al(static_cast<size_t>(axis * heads_kv) * kInfoBytes);
  L.off_zero = o;    o += kRowBytes;
  L.off_ranges = o;  o = al(o + static_cast<size_t>(2 * L.tiles) * 2 * sizeof(int32_t));
  L.off_part = o;    o = al(o + static_cast<size_t>(pairs * L.chunks) * kKeys * sizeof(float));
  L.bytes = o;
  return L;
}

}  // namespace
}  // namespace swattn

using namespace swattn;
using namespace swattn::tiles;

extern "C" {

size_t swattn_prefill_key_weights_workspace_bytes(int32_t batch, int64_t seq_kv, int32_t heads_q,
                                                  int32_t heads_kv, int32_t head_dim, int64_t n_full,
                                                  int64_t n_local) {
  if (batch < 1 || seq_kv < 1 || seq_kv > INT32_MAX || heads_q < 1 || heads_kv < 1 || heads_q % heads_kv ||
      head_dim != kD || n_full < 0 || n_local < 0 || n_full > INT32_MAX || n_local > INT32_MAX)
    return 0;
  return layout(batch * seq_kv, heads_kv, heads_q / heads_kv, n_full, n_local).bytes;
}

int swattn_prefill_key_weights(const void* q, const void* k, const float* lse,
                               const int32_t* full_idx, int64_t n_full, const int32_t* local_idx,
                               int64_t n_local, const int32_t* full_starts,
                               const int32_t* local_starts, const int32_t* causal_ends,
                               float* key_weights, int32_t batch, int64_t seq_q, int64_t seq_kv,
                               int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                               int32_t window, float scale_log2, void* workspace,
                               size_t workspace_bytes, void* stream) {
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
  const int64_t pairs = L.tiles * heads_kv, grid = pairs * L.chunks;
  const int64_t prep = ceil_div(L.blocks[0] + L.blocks[1], 8) * heads_kv, ranges = ceil_div(2 * L.tiles, kThreads / 64);
  if (grid > INT32_MAX || prep + ranges > INT32_MAX) return invalid(n + ": grid too large");
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
  p.zero_row = reinterpret_cast<uint16_t*>(ws + L.off_zero);
  p.ranges = reinterpret_cast<int32_t*>(ws + L.off_ranges);
  p.part = reinterpret_cast<float*>(ws + L.off_part);
  p.tiles = static_cast<int32_t>(L.tiles);
  p.chunk = static_cast<int32_t>(std::min<int64_t>(L.chunk, INT32_MAX / 2));
  p.chunks = static_cast<int32_t>(L.chunks);
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
  const dim3 gp(static_cast<uint32_t>(prep + ranges));
  if (meta)
    hipLaunchKernelGGL(weights_prep_kernel<true>, gp, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL(weights_prep_kernel<false>, gp, dim3(kThreads), 0, st, p);
  hipLaunchKernelGGL(weights_kernel, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), 0, st, p);
  hipLaunchKernelGGL(weights_reduce_kernel, dim3(static_cast<uint32_t>(pairs)), dim3(kThreads), 0, st, p);
  return launch_status(n.c_str());
}

}  // extern "C"
