// Routed GQA decode of sequences that continue shared prefixes, for gfx950
// (include/swattn_shared.h): the rule of swattn_decode.hip over a prefix's rows and then
// the sequence's own.  No counterpart in the reference.
//
//   s_j = c q.k_j,  p_j = 2^(s_j - m),  O = sum p_j v_j / sum p_j,  LSE = m + log2 sum p_j
//
// One launch takes both kinds of keys, a second merges their fp32 partials:
// * own rows: the line of routed (sequence, KV head) pairs that the decode over whole
//   caches shares out over workgroups (decode_line.h).  HBM-bound, with the products on
//   the matrix cores as in swattn_cache_decode.hip, so that the vector ALUs are free for
//   the prefixes.
// * prefixes: the query rows of all sequences that attend a prefix form tiles of up to
//   128 rows per KV head, full and local routes apart; a tile's keys are cut into pieces,
//   one per workgroup.  K and V are read once per tile, 64 keys at a time, into LDS
//   (global -> LDS DMA, double-buffered) and both products run on the matrix cores, a
//   wave per 32 rows: S^T = K Q^T, and O^T = V^T P^T with V transposed by the LDS
//   reads.  S^T's accumulator layout is P^T's operand layout.
// The first workgroups take prefix pieces, the others shares of the line; how many of
// each is settled on the device by every workgroup for itself, from the lengths.
//
// P enters its product as bf16 numbers: of a sequence's own rows three, 24 bits, as HBM is the limit
// there (B64 of 1024 rows behind 8192: 49.0 us with two, 49.5 with three); of a prefix two, its value and
// what that leaves, 17 bits (the prefill rounds P to one), as each is a third of a tile's matrix
// instructions: B64 Hq64 behind 32768 rows 131 us, with three 154, with one 17 less.  Of 524288
// outputs there 889 differ from the exact value's rounding, by one last place, with three 269,
// and 627 of a plain evaluation in fp32; behind 8192 rows 328 of 262144, 90 and 113.
//
// Local rows attend the last rows of their prefix only, each from its own start on.
// Masked scores are -inf, their weights 0.  A piece whose sums are not finite runs again
// carefully: values that are not finite, which a weight of 0 would turn into NaN, are
// taken out of the products and added key by key to the rows that attend them.
//
// Measured (Hkv 8), as a large copy's 5.2 TB/s and a large matrix product's 1210 TFLOP/s go:
// B64 Hq32 behind 8192 rows, own caches of 1024, a quarter full: 49.5 us against 39 for its bytes,
// own rows being read until 36 us of a split kernel of 45 (plan 2.2, merge and gap 7); B64 Hq64
// behind 32768 rows, all full: 131 to 134 us against 58 for its operations: the matrix cores are busy
// 48 % of the cycles and the vector ALUs 50 %, at 1.7 GHz, the two waves of a SIMD taking turns
// (a wave waits 28 % of its cycles for tiles and barriers, 34 % to issue).  Three documents, B40
// Hq40: 28.4 us against 19; B4 Hq8/Hkv2 behind 1024 rows 10.4 us, latency: plan, one tile, merge.
// Tried without gain: half tiles with operands read a step ahead (145 us instead of 134
// behind 32768 rows: more barriers), waves that share a short tile's keys and dims (such pieces
// wait for memory), unlike wave priorities.

#include <limits.h>
#include <math.h>

#include <string>

#include "decode_line.h"
#include "shared_plan.h"
#include "swattn_internal.h"
#include "swattn_shared.h"
#include "tiles.h"

namespace swattn {
namespace {

using tiles::bf16x8;
using tiles::f32x16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

static_assert(kTileKeys == tiles::kBN, "a step takes a tile of K");

constexpr int kOwnWaves = 4;         // waves per workgroup
constexpr int kMaxG = 8;
constexpr int kOwnStep = 32;         // keys that a wave takes at once of a sequence's own

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct SharedParams : DecodeCommon {
  static constexpr uint32_t kMinShare = 128;
  static constexpr uint32_t kLongShare = UINT32_MAX;
  static constexpr uint32_t kAlignSlack = 80;
  static constexpr bool kKeepNan = true;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* prefix_k;
  const uint16_t* prefix_v;
  const int32_t* prefix_lens;
  const int32_t* prefix_ids;
  float* tile_o;      // [piece][tile_rows][128] partials of prefix pieces
  float* tile_ml;     // [piece][tile_rows][2]
  int4* place;        // per sequence {first piece of KV head 0, pieces, first row, -}
  int prefixes, prefix_len;
  int tile_seqs;      // sequences of a tile, at most
  uint32_t tile_inv;  // 2^20 / tile_seqs, rounded up
  int tile_rows;      // rows that a partial has room for
  uint32_t target_inv;   // 2^32 / target, rounded up
  uint32_t least;     // workgroups that take the line, at least
  float c;            // sm_scale * log2(e)
  int stream_prefix;
};

__device__ __forceinline__ float bf(uint32_t bits16) { return __uint_as_float(bits16 << 16); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const bf16x2 x = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, x);
}
__device__ __forceinline__ int uniform(uint32_t x) {
  return static_cast<int>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}

// What a workgroup that takes a prefix piece has to know.
struct Piece {
  int group, tile, kvh, part;   // group = 2 * prefix + (local)
  int parts, length;            // pieces of a tile, keys of a piece
  int first, end;               // keys that the group's rows attend
  int seqs;                     // of the group
  int base;                     // the group's first piece
};

// A thread's sequences and prefixes: one of each, for up to 256 in a call, or four.  (The
// plan is straight-line code that every launch fetches anew: four 3.0 us, one 2.2.)
template <int kPer>
struct Routes {
  int group[kPer], start[kPer];   // group -1: attends no prefix row
  int lo[kPer], n[kPer];          // own rows
};

// The plan's LDS words of the prefixes: rows, sequences that attend them (routed full in the
// low 16 bits, local in the high ones), and the first key that a local one attends.
template <int kPer>
struct PrefixWords {
  int rows[256 * kPer];
  uint32_t seqs[256 * kPer];
  int first[256 * kPer];
};
constexpr int kMostPer = SWATTN_SHARED_MAX_PREFIXES / 256;
static_assert(kMostPer == kInlinePer && SWATTN_SHARED_MAX_SEQS == kInlineSeqs, "as many prefixes as sequences");

// What a thread's sequences attend; lengths, routes and prefixes are loaded at once.
template <int kPer>
__device__ __forceinline__ void routes_of(const SharedParams& p, int per, PrefixWords<kPer>& s, Routes<kPer>& r) {
  int id[kPer];
  bool full[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int b = static_cast<int>(threadIdx.x) * per + j;
    id[j] = -1;
    full[j] = false;
    r.lo[j] = r.n[j] = 0;
    if (j >= per || b >= p.batch) continue;
    key_range(p, b, r.lo[j], r.n[j]);
    id[j] = p.prefix_ids[b];
    full[j] = p.full[b] != 0;
  }
  for (int i = threadIdx.x; i < p.prefixes; i += 256) {
    s.rows[i] = min(max(p.prefix_lens[i], 0), p.prefix_len);
    s.seqs[i] = 0;
    s.first[i] = INT_MAX;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    r.group[j] = -1;
    r.start[j] = 0;
    if (id[j] < 0 || id[j] >= p.prefixes) continue;
    const int rows = s.rows[id[j]], len = r.lo[j] + r.n[j];
    r.start[j] = prefix_start(full[j], rows, len, p.window);
    if (r.start[j] >= rows) continue;
    r.group[j] = 2 * id[j] + (full[j] ? 0 : 1);
    atomicAdd(&s.seqs[id[j]], full[j] ? 1u : 1u << 16);
    if (!full[j]) atomicMin(&s.first[id[j]], r.start[j]);
  }
}

// The workgroup's part: a prefix piece (true), or a share of the line (false; st.take 0
// past its end).
template <int kPer>
__device__ __forceinline__ bool plan_shared(const SharedParams& p, const Routes<kPer>& r, int per, const PrefixWords<kPer>& s,
                                            SeqEntry* s_ent, Piece& piece, SplitStart& st, uint32_t& wg) {
  __shared__ Piece s_piece;
  __shared__ SplitStart s_start;
  const int tid = threadIdx.x;
  uint32_t keys = 0, cnt = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    keys += r.n[j];
    cnt += r.n[j] > 0 ? 1 : 0;
  }
  uint32_t before, rank, all_keys, all_cnt;
  scan_keys<4, 0, uint32_t>(keys, cnt, before, rank, all_keys, all_cnt);   // (its barrier orders the atomics too)
  const uint32_t line = (all_keys + all_cnt * p.pad) * p.hkv;
  // This thread's groups, (prefix, route), in order: sequences, tiles, keys.
  const int pper = kPer == 1 ? 1 : (p.prefixes + 255) >> 8;
  struct Group {
    uint32_t seqs, tiles, first, keys;
  };
  Group g[2 * kPer];
  uint32_t positions = 0, all_positions, unused0, unused1, unused2;
#pragma unroll
  for (int i = 0; i < 2 * kPer; ++i) {
    const int x = tid * pper + i / 2;
    g[i] = Group{0, 0, 0, 0};
    if (i / 2 >= pper || x >= p.prefixes) continue;
    g[i].seqs = i & 1 ? s.seqs[x] >> 16 : s.seqs[x] & 0xffffu;
    if (g[i].seqs == 0) continue;
    g[i].tiles = tiles_of(g[i].seqs, p.tile_seqs, p.tile_inv);
    g[i].first = i & 1 ? s.first[x] : 0;
    g[i].keys = static_cast<uint32_t>(s.rows[x]) - g[i].first;
    positions += g[i].tiles * g[i].keys;
  }
  scan_keys<4, 1, uint32_t>(positions, 0, unused0, unused1, all_positions, unused2);
  const uint32_t length = piece_length(line, all_positions, p.hkv, p.target_inv, p.prefix_len);
  uint32_t pieces = 0, base, all_pieces, parts[2 * kPer], len[2 * kPer];
#pragma unroll
  for (int i = 0; i < 2 * kPer; ++i) {
    parts[i] = len[i] = 0;
    if (g[i].seqs == 0) continue;
    const Cut cut = cut_keys(g[i].keys, length);
    len[i] = cut.length;
    parts[i] = cut.parts;
    pieces += g[i].tiles * p.hkv * parts[i];
  }
  scan_keys<4, 2, uint32_t>(pieces, 0, base, unused0, all_pieces, unused1);
  const uint32_t block = blockIdx.x;
  if (block < all_pieces) {   // uniform
    if (block - base < pieces) {
#pragma unroll
      for (int i = 0; i < 2 * kPer; ++i) {
        const uint32_t here = g[i].tiles * p.hkv * parts[i];
        if (block - base < here) {
          const PieceOf x = piece_of(block - base, here, g[i].tiles, parts[i]);
          s_piece = Piece{2 * (tid * pper + i / 2) + (i & 1), static_cast<int>(x.tile), static_cast<int>(x.kvh),
                          static_cast<int>(x.part), static_cast<int>(parts[i]), static_cast<int>(len[i]),
                          static_cast<int>(g[i].first), static_cast<int>(g[i].first + g[i].keys), static_cast<int>(g[i].seqs),
                          static_cast<int>(base)};
        }
        base += here;
      }
    }
    __syncthreads();
    piece = s_piece;
    return true;
  }
  // The line, as plan_inline lays it out for the workgroups that the pieces leave.
  wg = block - all_pieces;
  SharedParams q = p;
  q.target = line_target(p.target, all_pieces, p.least);
  Line<uint32_t> L = plan_line<uint32_t>(q, all_keys * p.hkv, all_cnt * p.hkv);
  before += rank * p.pad;
  if (L.aligned) {
    uint32_t len = 0, none;
#pragma unroll
    for (int j = 0; j < kPer; ++j) len += L.length(r.n[j], 0);
    scan_keys<4, 3, uint32_t>(len, 0, before, none, L.total, none);
    L.total *= p.hkv;
  }
  const uint64_t pos64 = static_cast<uint64_t>(wg) * L.share;
  const uint32_t pos = static_cast<uint32_t>(min(pos64, static_cast<uint64_t>(L.total)));
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int b = tid * per + j;
    const uint32_t off = before * p.hkv, len = L.length(r.n[j], p.pad);
    if (wg == 0 && j < per && b < p.batch) {
      p.plan[1 + b] = plan_entry(off, r.n[j], rank, len);
      if (r.group[j] < 0) p.place[b] = make_int4(0, 0, 0, 0);
    }
    if (r.n[j] > 0) {
      s_ent[rank] = SeqEntry{b, r.lo[j], r.n[j], len};
      if (pos >= off && pos - off < len * p.hkv) split_start(s_start, rank, pos - off, len);
      ++rank;
    }
    before += len;
  }
  if (wg == 0 && tid == 0) p.plan[0] = make_uint4(L.share, L.total, 0u, UINT32_MAX / L.share);
  st.take = 0;
  if (pos >= L.total) return false;   // uniform
  __syncthreads();
  st = s_start;
  st.take = min(L.total - pos, L.share);
  return false;
}

// 64 keys of K and V as LDS tiles [64][128], 16-byte chunks swizzled by tiles::swz: wave w
// copies rows 16 w .. 16 w + 15 of both, four rows per instruction; rows behind `last` are
// read as that one.
constexpr int kSlotBytes = 2 * tiles::kTileBytes;
__device__ __forceinline__ void copy_tile(const uint16_t* kb, const uint16_t* vb, uint32_t row_bytes, int key, int last,
                                          uint32_t lds, int wave, int lane, bool stream) {
  const int64_t at = static_cast<int64_t>(key + 16 * wave) * (row_bytes / 2);
  const uint32_t chunk = 16u * ((lane & 15) ^ ((lane >> 4) << 2));   // of row 4 i + lane / 16: ^ 16 i
  uint32_t row = (lane >> 4) * row_bytes;   // a tile's rows span less than 2^31 bytes
  lds += 4096u * static_cast<uint32_t>(wave);
  if (key + kTileKeys - 1 <= last) {   // uniform
    auto whole = [&](auto dma) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t to = at + static_cast<int64_t>(4 * i) * (row_bytes / 2);
        const uint32_t off = (chunk ^ (16u * i)) + row;
        dma(kb + to, off, lds + 1024u * i);
        dma(vb + to, off, lds + 1024u * i + tiles::kTileBytes);
      }
    };
    if (stream)   // uniform
      whole([](const void* from, uint32_t off, uint32_t to) { tiles::dma16_stream_from(from, off, to); });
    else
      whole([](const void* from, uint32_t off, uint32_t to) { tiles::dma16_from(from, off, to); });
  } else {
    const int rest = last - key - 16 * wave;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Rows count from the wave's first, or back from it to the last one.
      const int64_t off = static_cast<int64_t>(min(4 * i + (lane >> 4), rest)) * static_cast<int64_t>(row_bytes) + (chunk ^ (16u * i));
      tiles::dma16_gather(reinterpret_cast<const char*>(kb + at) + off, lds + 1024u * i);
      tiles::dma16_gather(reinterpret_cast<const char*>(vb + at) + off, lds + 1024u * i + tiles::kTileBytes);
    }
  }
}

__device__ __forceinline__ bool odd_pair(uint32_t x) {   // whether one of two bf16 numbers is not finite
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

// A wave's 32 rows: lane (r, h) = (lane % 32, lane / 32) has row r, keys 8 j + 4 h + i of
// each 32 and dims 32 d + 8 j + 4 h + i.
struct RowState {
  float m, l;        // maximum (the same in both lanes of a row); this lane's share of the sum
  f32x16 acc[4];
};

// Where a lane's operands lie in a tile of K and one of V, from LDS address 0: a chunk's
// number enters by XOR, the rest of a row's place is added.
struct LaneLds {
  uint32_t k;   // key r of K, dims 8 h .. +7; ^ 32 d: those of dims 16 d, + 8192 f: key 32 f + r
  uint32_t v;   // V^T operand: ^ (64 d + 32 x): dims 32 d, + 256 (32 f + 16 t + 8 x): keys of group t, half x
};
__device__ __forceinline__ LaneLds lane_lds(uint32_t ring, int lane) {
  const int r = lane & 31, h = lane >> 5, half = (lane >> 4) & 1, i = lane & 15;
  return LaneLds{ring + tiles::kRowBytes * r + 16 * (h ^ tiles::swz(r)),
                 ring + tiles::kTileBytes + tiles::kRowBytes * (4 * h + (i >> 2)) +
                     16 * ((2 * half + ((i & 3) >> 1)) ^ (((i >> 2) << 2) | h)) + 8 * (i & 1)};
}
// The places in slot `slot` of the ring, made anew for each tile: kept, the XORed ones take
// registers that the loop does not have.
__device__ __forceinline__ LaneLds in_slot(LaneLds at, uint32_t slot) {
  at.k += slot;
  at.v += slot;
  asm volatile("" : "+v"(at.k), "+v"(at.v));
  return at;
}
typedef __attribute__((address_space(3))) const bf16x8* LdsChunk;
typedef __attribute__((address_space(3))) s16x4* LdsFour;

// Scheduling groups (__builtin_amdgcn_sched_group_barrier).
constexpr int kValu = 0x2, kMfma = 0x8, kLdsRead = 0x100, kTrans = 0x400;

// A group of 16 keys of V^T, all 128 dims.
struct VGroup {
  uint32_t x[4][4];   // [32 dims][operand]
};
__device__ __forceinline__ void read_v(const LaneLds& at, int group, int d, VGroup& v) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (LdsFour)(uintptr_t)((at.v ^ (64 * d + 32 * x)) + (16 * group + 8 * x) * tiles::kRowBytes));
    const uint2 two = __builtin_bit_cast(uint2, four);
    v.x[d][2 * x] = two.x;
    v.x[d][2 * x + 1] = two.y;
  }
}

// 8 weights of a group of 16 keys, as the two operands of their products.
struct PGroup {
  u32x4 hi, lo;
};
__device__ __forceinline__ PGroup split_p(const float (&y)[8]) {
  PGroup p;
#pragma unroll
  for (int e = 0; e < 4; ++e) {   // the differences are exact
    p.hi[e] = pack2(y[2 * e], y[2 * e + 1]);
    p.lo[e] = pack2(y[2 * e] - __uint_as_float(p.hi[e] << 16), y[2 * e + 1] - __uint_as_float(p.hi[e] & 0xffff0000u));
  }
  return p;
}

// 32 keys f of a tile: S^T = K Q^T.
__device__ __forceinline__ f32x16 scores(const LaneLds& at, int f, const bf16x8 (&q)[8]) {
  f32x16 s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const bf16x8 a = *(LdsChunk)(uintptr_t)((at.k ^ (32 * d)) + 32 * f * tiles::kRowBytes);
    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[d], s, 0, 0, 0);
  }
  return s;
}

// Moves the rows' maxima where a score exceeds one by more than 8 in the exp2 domain (rare);
// top: this lane's largest raw score.  Returns what weights are taken from: the maximum, 0
// where there were only scores of -inf so far, which then weigh nothing.
__device__ __forceinline__ float move_maxima(float top, float c, RowState& w) {
  top *= c;
  if (__builtin_amdgcn_ballot_w64(top - w.m > 8.0f)) {
    top = tiles::xor32_max(top);
    const float mn = top - w.m > 8.0f ? top : w.m;
    const float a = mn == w.m ? 1.0f : __builtin_amdgcn_exp2f(w.m - mn);
    w.m = mn;
    w.l *= a;
#pragma unroll
    for (int d = 0; d < 4; ++d) w.acc[d] *= a;
  }
  return w.m == -INFINITY ? 0.f : w.m;
}

// Scores of keys that a row does not attend become -inf: it attends `count` of them from
// number `first` of the tile on (counted from this lane's first key, 4 h).
__device__ __forceinline__ void mask(f32x16 (&s)[2], int first, uint32_t count) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int at = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3);
    if (static_cast<uint32_t>(at - first) >= count) s[i >> 4][i & 15] = -INFINITY;
  }
}

// 64 keys; kMask: of which rows do not attend all.  The weights of the next 16 keys are
// made, and their V read, under the products of the last ones.
template <bool kMask>
__device__ __forceinline__ void tile_step(const LaneLds& at, const bf16x8 (&q)[8], float c, int first, uint32_t count, RowState& w) {
  f32x16 s[2] = {scores(at, 0, q), scores(at, 1, q)};
  VGroup v;
#pragma unroll
  for (int d = 0; d < 4; ++d) read_v(at, 0, d, v);
  __builtin_amdgcn_sched_group_barrier(kLdsRead, 4, 0);
#pragma unroll
  for (int i = 0; i < 12; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kLdsRead, 1, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kLdsRead, 2, 0);
  }
  if (kMask) mask(s, first, count);
  float top = s[0][0];
#pragma unroll
  for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
  const float from = move_maxima(top, c, w);
  auto weights = [&](int g) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + i], c, -from));
      w.l += y[i];
    }
    return split_p(y);
  };
  PGroup p = weights(0);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    asm volatile("" : "+v"(p.hi), "+v"(p.lo));
    __builtin_amdgcn_sched_barrier(0);
    PGroup next = p;
    if (g < 3) next = weights(g + 1);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const bf16x8 a = __builtin_bit_cast(bf16x8, v.x[d]);
      w.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, p.hi), w.acc[d], 0, 0, 0);
      w.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, p.lo), w.acc[d], 0, 0, 0);
      if (g < 3) read_v(at, g + 1, d, v);
    }
    p = next;
    if (g < 3) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kLdsRead, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kValu, 4, 0);
        __builtin_amdgcn_sched_group_barrier(kTrans, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kValu, 3, 0);
      }
    }
  }
}

// The same where values are not finite, which a weight of 0 does not keep out, and of which
// an infinite one times a weight's second part can make NaN: the products go without them,
// and they are added key by key to the rows that attend them.  vt: the tile of V.
__device__ __forceinline__ void careful_step(const char* vt, const LaneLds& at_lds, const bf16x8 (&q)[8], float c, int first,
                                             uint32_t count, RowState& w, int lane) {
  const int h = lane >> 5;
  f32x16 s[2] = {scores(at_lds, 0, q), scores(at_lds, 1, q)};
  mask(s, first, count);
  float top = s[0][0];
#pragma unroll
  for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
  const float from = move_maxima(top, c, w);
  bool odd = false;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = 8 * (g & 1) + i;
      y[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][x], c, -from));
      w.l += y[i];
      s[g >> 1][x] = y[i];
    }
    const PGroup p = split_p(y);
    VGroup v;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      read_v(at_lds, g, d, v);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t& u = v.x[d][x];
        odd = odd || odd_pair(u);
        if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
        if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
      }
      w.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v.x[d]), __builtin_bit_cast(bf16x8, p.hi), w.acc[d], 0, 0, 0);
      w.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v.x[d]), __builtin_bit_cast(bf16x8, p.lo), w.acc[d], 0, 0, 0);
    }
  }
  if (__builtin_amdgcn_ballot_w64(odd) == 0) return;
  // Values that are not finite, key by key: what they add to the rows that attend them.
  for (int at = 0; at < kTileKeys; ++at) {
    const char* row = vt + at * tiles::kRowBytes;
    const uint32_t mine = *reinterpret_cast<const uint32_t*>(row + 16 * ((lane >> 2) ^ tiles::swz(at)) + 4 * (lane & 3));
    if (__builtin_amdgcn_ballot_w64(odd_pair(mine)) == 0) continue;
    float pr = 0.f;   // the weight, in the lane whose keys it is among
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (at >> 5 == f && ((at >> 3) & 3) == i >> 2 && (at & 3) == (i & 3)) pr = s[f][i];
    const float other = __shfl_xor(pr, 32);
    if (((at >> 2) & 1) != h) pr = other;
    if (static_cast<uint32_t>(at - 4 * h - first) >= count) continue;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int dim = 32 * d + 8 * (i >> 2) + 4 * h + (i & 3);
        const uint32_t bits = *reinterpret_cast<const uint16_t*>(row + 16 * ((dim >> 3) ^ tiles::swz(at)) + 2 * (dim & 7));
        if ((bits & 0x7f80u) == 0x7f80u) w.acc[d][i] += pr * bf(bits);
      }
  }
}

// One workgroup: piece `part` of a tile's keys, for KV head kvh.
template <int kPer>
__device__ __forceinline__ void prefix_piece(const SharedParams& p, const Routes<kPer>& routes, int per, const Piece& x,
                                             int2* s_rows, char* ring) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int k0 = uniform(x.first + x.part * x.length), k1 = k0 + min(uniform(x.length), uniform(x.end) - k0);
  const uint32_t row_bytes = static_cast<uint32_t>(p.hkv) * tiles::kRowBytes;
  const int64_t base = (static_cast<int64_t>(uniform(x.group) >> 1) * p.prefix_len * p.hkv + uniform(x.kvh)) * kD;
  const int last = uniform(x.end) - 1;
  const uint16_t *kb = p.prefix_k + base, *vb = p.prefix_v + base;
  const uint32_t lds = tiles::lds_addr(ring);
  const int steps = (k1 - k0 + kTileKeys - 1) / kTileKeys;
  auto copy = [&](int j) {
    copy_tile(kb, vb, row_bytes, k0 + kTileKeys * j, last, lds + (j & 1) * kSlotBytes, wave, lane, p.stream_prefix != 0);
  };
  auto copy_first = [&]() {
    copy(0);
    if (steps > 1) copy(1);
  };
  copy_first();
  // The tile's sequences, in order.
  uint32_t cnt = 0, rank, unused0, unused1, unused2;
#pragma unroll
  for (int j = 0; j < kPer; ++j) cnt += routes.group[j] == x.group ? 1 : 0;
  scan_keys<4, 4, uint32_t>(0, cnt, unused0, rank, unused1, unused2);
  const int first_seq = x.tile * p.tile_seqs, seqs = min(x.seqs - first_seq, p.tile_seqs);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (routes.group[j] != x.group) continue;
    const int at = static_cast<int>(rank++) - first_seq, b = tid * per + j;
    if (at < 0 || at >= seqs) continue;
    s_rows[at] = make_int2(b, routes.start[j]);
    if (x.kvh == 0 && x.part == 0)
      p.place[b] = make_int4(x.base + x.tile * p.hkv * x.parts, x.parts, at * p.group, 0);
  }
  __syncthreads();   // the rows
  // This lane's row.
  const int rows = seqs * p.group, row = 32 * wave + (lane & 31), h = lane >> 5;
  const bool mine = row < rows, busy = 32 * wave < rows;   // busy: uniform
  const int seq = min(row, rows - 1) / p.group;
  const int2 entry = s_rows[seq];
  const int64_t at = static_cast<int64_t>(entry.x) * p.hq + x.kvh * p.group + (min(row, rows - 1) - seq * p.group);
  bf16x8 q[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    u32x4 u = *reinterpret_cast<const u32x4*>(p.q + at * kD + 16 * d + 8 * h);
    if (p.c < 0.f) u ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};   // so that a score's scale is positive
    if (!mine) u = u32x4{0, 0, 0, 0};
    q[d] = __builtin_bit_cast(bf16x8, u);
  }
  const float c = fmaxf(fabsf(p.c), 0x1p-126f);   // not 0, which would make NaN of masked scores
  const int start = entry.y, latest = __builtin_amdgcn_readfirstlane(tiles::wave_max(start));
  const LaneLds at_lds = lane_lds(lds, lane);
  RowState w;
  // Once, and carefully if a sum is not finite then.
  for (int careful = 0; careful < 2; ++careful) {
    w.m = -INFINITY;
    w.l = 0.f;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) w.acc[d][i] = 0.f;
    // Tiles that some row attends in part (they start later), whole ones, the ragged end.
    const int head = min(max((latest - k0 + kTileKeys - 1) / kTileKeys, 0), steps);
    const int tail = max(k1 - k0 == steps * kTileKeys ? steps : steps - 1, head);
    int j = 0;
    auto arrive = [&]() {   // tile j is there, and every wave is done with the one before
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (j > 0 && j + 1 < steps) copy(j + 1);
      return static_cast<uint32_t>(j & 1) * kSlotBytes;
    };
    // What this row attends of tile j.
    auto from = [&]() { return max(start - (k0 + kTileKeys * j), 0) - 4 * h; };
    auto count = [&]() {
      const int key = k0 + kTileKeys * j;
      return static_cast<uint32_t>(max(min(k1 - key, kTileKeys) - max(start - key, 0), 0));
    };
    auto masked = [&]() {
      const LaneLds at = in_slot(at_lds, arrive());
      if (busy) tile_step<true>(at, q, c, from(), count(), w);
    };
    if (careful) {
      for (; j < steps; ++j) {
        const uint32_t slot = arrive();
        if (busy) careful_step(ring + slot + tiles::kTileBytes, in_slot(at_lds, slot), q, c, from(), count(), w, lane);
      }
      break;
    }
    for (; j < head; ++j) masked();
    if (busy) {
      for (; j < tail; ++j) tile_step<false>(in_slot(at_lds, arrive()), q, c, 0, 0, w);
    } else {
      for (; j < tail; ++j) arrive();
    }
    for (; j < steps; ++j) masked();
    float sum = 0.f;   // not finite if one of them is not
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(w.acc[d][i], 0.f, sum);
    if (!__syncthreads_or(mine && sum != 0.f)) break;
    copy_first();
  }
  if (!mine) return;
  w.l = w.l + __shfl_xor(w.l, 32);
  const int64_t to = static_cast<int64_t>(x.base + (x.tile * p.hkv + x.kvh) * x.parts + x.part) * p.tile_rows + row;
  if (h == 0) *reinterpret_cast<float2*>(p.tile_ml + 2 * to) = make_float2(w.m, w.l);
  float* o = p.tile_o + to * kD + 4 * h;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(o + 32 * d + 8 * j) =
          make_float4(w.acc[d][4 * j], w.acc[d][4 * j + 1], w.acc[d][4 * j + 2], w.acc[d][4 * j + 3]);
}

// One partial (maximum, sum, unnormalised output) per wave and head.
struct PieceLds {
  float m[kOwnWaves][kMaxG], l[kOwnWaves][kMaxG];
  float acc[kOwnWaves][kMaxG][kD];
};

// The partials of keys [k0, k1) with one key per wave at a time on the vector ALUs: where
// the products met values that are not finite.  A weight is one fp32 number here, so that
// an infinite value stays infinite, and nothing but the piece's rows is read.
__device__ __forceinline__ void careful_piece(const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t stride,
                                              int k0, int k1, int group, float c, int wave, int lane,
                                              PieceLds& lds) {
  for (int h = 0; h < group; ++h) {
    const uint32_t qx = *reinterpret_cast<const uint32_t*>(q + h * kD + 2 * lane);
    float m = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
    for (int key = k0 + wave; key < k1; key += kOwnWaves) {
      const uint32_t kx = *reinterpret_cast<const uint32_t*>(k + key * stride + 2 * lane);
      const uint32_t vx = *reinterpret_cast<const uint32_t*>(v + key * stride + 2 * lane);
      const float s = c * wave_all(__builtin_fmaf(bf(qx >> 16), bf(kx >> 16), bf(qx & 0xffffu) * bf(kx & 0xffffu)), Add());
      if (s > m) {
        const float a = __builtin_amdgcn_exp2f(m - s);
        l *= a;
        a0 *= a;
        a1 *= a;
        m = s;
      }
      const float pr = __builtin_amdgcn_exp2f(s - (m == -INFINITY ? 0.f : m));
      l += pr;
      a0 += pr * bf(vx & 0xffffu);
      a1 += pr * bf(vx >> 16);
    }
    *reinterpret_cast<float2*>(&lds.acc[wave][h][2 * lane]) = make_float2(a0, a1);
    if (lane == 0) {
      lds.m[wave][h] = m;
      lds.l[wave][h] = l;
    }
  }
}

template <bool kStream>
__device__ __forceinline__ u32x4 load16(const uint16_t* p) {
  const u32x4* at = reinterpret_cast<const u32x4*>(p);
  return kStream ? __builtin_nontemporal_load(at) : *at;
}

// One share of the line: its pairs one after the other, a piece of each.  A wave takes 32
// keys at once, steps w, w + 4, ... of a piece; rows outside it are read as its nearest
// row and masked.
// * S^T [16 keys x 16 columns] = K Q^T, v_mfma_f32_16x16x32_bf16: lane (c, g) = (lane % 16,
//   lane / 16) holds key c of the tile, dims 32 j + 8 g .. +7; column c is head c % 8.
// * O^T [16 dims x 16 columns] += V^T P^T, 32 keys at once: lane (c, g) holds dims 8 c .. +7
//   of keys 4 g .. +3 of both key tiles; tile n takes dim 8 c + n of each, so that S^T's
//   accumulator layout is P^T's operand layout, and V is transposed inside a lane.
//   A weight enters as three bf16 numbers, 24 bits: columns 0-7 take the first in one product
//   and the third in a second, columns 8-15 the one between.
// A piece's partial lies in slot wg + (pair's rank): both only grow along the line, one of
// them at every step from piece to piece, so that no two pieces share a slot and a pair's
// slots are consecutive.
template <bool kStream>
__device__ __forceinline__ void own_pieces(const SharedParams& p, uint32_t wg, const SplitStart& st, const SeqEntry* s_ent,
                                           PieceLds& lds) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  int r = uniform(st.r), kvh = uniform(st.kvh);
  uint32_t key = uniform(st.key);
  uint32_t left = uniform(st.take);
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, g = lane >> 4, G = p.group, head = c & 7;
  const bool second = c >= 8;
  const int64_t stride = static_cast<int64_t>(p.hkv) * kD;
  for (;;) {
    const SeqEntry e = s_ent[r];
    const int b = uniform(e.b);
    const uint32_t n = uniform(e.n), len = uniform(e.len);
    const uint32_t took = min(left, len - key);
    left -= took;
    if (key < n) {   // else this share starts in the pair's padding
      const int64_t slot = static_cast<int64_t>(wg) + static_cast<int64_t>(r) * p.hkv + kvh;
      const int k0 = uniform(e.lo) + static_cast<int>(key), k1 = k0 + static_cast<int>(min(took, n - key));
      const uint16_t* qb = p.q + (static_cast<int64_t>(b) * p.hq + kvh * G) * kD;
      const int64_t base = static_cast<int64_t>(b) * p.cache_len * stride + kvh * kD;
      const uint16_t *kb = p.k + base + 8 * g, *vb = p.v + base + 8 * c;
      bf16x8 q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 u = *reinterpret_cast<const u32x4*>(qb + min(head, G - 1) * kD + 32 * j + 8 * g);
        if (head >= G) u = u32x4{0, 0, 0, 0};
        q[j] = __builtin_bit_cast(bf16x8, u);
      }
      const int steps = (k1 - k0 + kOwnStep - 1) / kOwnStep;
      u32x4 kr[2][4], vr[8];
      auto load = [&](int i) {
        const int at = k0 + kOwnStep * i;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint16_t* row = kb + min(at + 16 * t + c, k1 - 1) * stride;
#pragma unroll
          for (int j = 0; j < 4; ++j) kr[t][j] = load16<kStream>(row + 32 * j);
        }
#pragma unroll
        for (int t = 0; t < 8; ++t)
          vr[t] = load16<kStream>(vb + min(at + 16 * (t >> 2) + 4 * g + (t & 3), k1 - 1) * stride);
      };
      load(wave);
      float m = -INFINITY, l = 0.f;   // column c's maximum, and this lane's share of its sum
      f32x4 acc[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int i = wave; i < steps; i += kOwnWaves) {
        const int at = k0 + kOwnStep * i;
        f32x4 s[2];
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[t][j]), q[j], s[t], 0, 0, 0);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            s[t][x] = at + 16 * t + 4 * g + x < k1 ? s[t][x] * p.c : -INFINITY;
            top = fmaxf(top, s[t][x]);
          }
        }
        if (__builtin_amdgcn_ballot_w64(top - m > 8.0f)) {   // rare: move the maxima, rescale
          top = with_lane32(with_lane16(top, Max()), Max());
          const float mn = top - m > 8.0f ? top : m;
          const float a = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= a;
#pragma unroll
          for (int t = 0; t < 8; ++t) acc[t] *= a;
        }
        const float from = m == -INFINITY ? 0.f : m;   // only scores of -inf so far: they weigh nothing
        u32x4 pk, pk2;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 4; x += 2) {
            float y[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              y[u] = __builtin_amdgcn_exp2f(s[t][x + u] - from);   // 0 behind the piece
              l += y[u];
            }
            const uint32_t high = pack2(y[0], y[1]);   // the differences are exact
            y[0] -= __uint_as_float(high << 16);
            y[1] -= __uint_as_float(high & 0xffff0000u);
            const uint32_t mid = pack2(y[0], y[1]);
            y[0] -= __uint_as_float(mid << 16);
            y[1] -= __uint_as_float(mid & 0xffff0000u);
            pk[2 * t + x / 2] = second ? mid : high;
            pk2[2 * t + x / 2] = second ? 0u : pack2(y[0], y[1]);
          }
        const bf16x8 pb = __builtin_bit_cast(bf16x8, pk), pb2 = __builtin_bit_cast(bf16x8, pk2);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          u32x4 a0, a1;   // dims 2 d and 2 d + 1 of this lane's eight
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            a0[t] = __builtin_amdgcn_perm(vr[2 * t + 1][d], vr[2 * t][d], 0x05040100u);
            a1[t] = __builtin_amdgcn_perm(vr[2 * t + 1][d], vr[2 * t][d], 0x07060302u);
          }
          acc[2 * d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), pb, acc[2 * d], 0, 0, 0);
          acc[2 * d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), pb, acc[2 * d + 1], 0, 0, 0);
          acc[2 * d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), pb2, acc[2 * d], 0, 0, 0);
          acc[2 * d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), pb2, acc[2 * d + 1], 0, 0, 0);
        }
        load(i + kOwnWaves);   // past the end: the last row, never used
      }
      // This wave's partial: column c's sum over its four lanes, O^T with its second
      // columns.  acc[t][x]: dim 8 (4 g + x) + t of column c.
      l = with_lane32(with_lane16(l, Add()), Add());
      float sum = 0.f;   // not 0 if one of the outputs is not finite
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          acc[t][x] += __shfl_xor(acc[t][x], 8);
          sum = __builtin_fmaf(acc[t][x], 0.f, sum);
        }
      if (c < G) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int t = 0; t < 8; t += 4)
            *reinterpret_cast<f32x4*>(&lds.acc[wave][c][8 * (4 * g + x) + t]) =
                f32x4{acc[t][x], acc[t + 1][x], acc[t + 2][x], acc[t + 3][x]};
        if (g == 0) {
          lds.m[wave][c] = m;
          lds.l[wave][c] = l;
        }
      }
      if (__syncthreads_or(sum != 0.f)) {
        careful_piece(qb, p.k + base, p.v + base, stride, k0, k1, G, p.c, wave, lane, lds);
        __syncthreads();
      }
      // Combine the waves: one partial per head.  Where no maximum is finite the sums are 0
      // or NaN, and stay.
      float* po = p.part_o + slot * G * kD;
      float* pml = p.part_ml + slot * G * 2;
      auto combine = [&](int h, auto of) {
        float mm = -INFINITY, x = 0.f;
#pragma unroll
        for (int w = 0; w < kOwnWaves; ++w) mm = fmaxf(mm, lds.m[w][h]);
#pragma unroll
        for (int w = 0; w < kOwnWaves; ++w) x += (mm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(lds.m[w][h] - mm)) * of(w);
        return make_float2(mm, x);
      };
      for (int i = tid; i < G * kD; i += 256) po[i] = combine(i / kD, [&](int w) { return lds.acc[w][i / kD][i & (kD - 1)]; }).y;
      if (tid < G) *reinterpret_cast<float2*>(pml + 2 * tid) = combine(tid, [&](int w) { return lds.l[w][tid]; });
    }
    // The rest of the share continues at the start of the next pair.
    if (left == 0u) return;
    key = 0;
    if (++kvh == p.hkv) {
      kvh = 0;
      ++r;
    }
    __syncthreads();   // the next piece's partials lie in the same LDS
  }
}

// A line share's entries and partials, or a ring of two tiles of K and V.
constexpr int kPieceOffset = kInlineSeqs * static_cast<int>(sizeof(SeqEntry));
constexpr int kLdsBytes = 2 * kSlotBytes;
static_assert(kPieceOffset + sizeof(PieceLds) <= kLdsBytes, "a share's words fit the ring");

template <int kPer, bool kStream>
__global__ __launch_bounds__(256, 2) void shared_split_kernel(const SharedParams p) {
  __shared__ __align__(1024) char s_mem[kLdsBytes];
  __shared__ PrefixWords<kPer> s_prefix;
  __shared__ int2 s_rows[kTileRows];
  const int per = kPer == 1 ? 1 : (p.batch + 255) >> 8;
  Routes<kPer> routes;
  routes_of(p, per, s_prefix, routes);
  Piece piece;
  SplitStart st;
  uint32_t wg = 0;
  SeqEntry* ent = reinterpret_cast<SeqEntry*>(s_mem);
  if (plan_shared(p, routes, per, s_prefix, ent, piece, st, wg))
    prefix_piece(p, routes, per, piece, s_rows, s_mem);
  else if (st.take > 0)
    own_pieces<kStream>(p, wg, st, ent, *reinterpret_cast<PieceLds*>(s_mem + kPieceOffset));
}

// One workgroup of 256 threads per output row: merge_row over the row's shares of the line
// and its prefix pieces, up to 256 of each.
__global__ __launch_bounds__(256) void shared_merge_kernel(const SharedParams p) {
  __shared__ float s_w[2 * kMaxSplitsDev];
  __shared__ float s_red[8];
  __shared__ float4 s_part[8][kD / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int64_t row = static_cast<int64_t>(b) * p.hq + kvh * p.group + h;
  const SeqPlace seq = seq_place(p.plan[1 + b]);
  const uint4 line = p.plan[0];
  const int4 place = p.place[b];
  const uint32_t off = static_cast<uint32_t>(seq.off) + static_cast<uint32_t>(kvh) * seq.len;
  const uint32_t wg0 = share_of(off, line.x, line.w);
  const int own = seq.n > 0 ? static_cast<int>(share_of(off + seq.n - 1, line.x, line.w) - wg0) + 1 : 0;   // at most 256
  const int pieces = place.y, all = own + pieces;
  const int64_t slot0 = static_cast<int64_t>(wg0) + static_cast<int64_t>(seq.rank) * p.hkv + kvh;
  const int64_t row0 = (static_cast<int64_t>(place.x) + static_cast<int64_t>(kvh) * pieces) * p.tile_rows + place.z + h;
  const int g = tid >> 5, q = tid & 31;
  auto part = [&](int c) -> const float4* {
    const float* at = c < own ? p.part_o + ((slot0 + c) * p.group + h) * kD
                              : p.tile_o + (row0 + static_cast<int64_t>(c - own) * p.tile_rows) * kD;
    return reinterpret_cast<const float4*>(at) + q;
  };
  float2 ml[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
  if (tid < own) ml[0] = *reinterpret_cast<const float2*>(p.part_ml + ((slot0 + tid) * p.group + h) * 2);
  if (tid < pieces) ml[1] = *reinterpret_cast<const float2*>(p.tile_ml + (row0 + static_cast<int64_t>(tid) * p.tile_rows) * 2);
  float4 ahead[kMergeAhead];
#pragma unroll
  for (int i = 0; i < kMergeAhead; ++i) {
    ahead[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g + 8 * i < all) ahead[i] = *part(g + 8 * i);
  }
  float mx = wave_all(fmaxf(ml[0].x, ml[1].x), Max());
  if (lane == 0) s_red[wave] = mx;
  __syncthreads();
  const float M = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  // Weights 2^(m - M); where no maximum is finite the sums are 0 or NaN, and stay.
  float wt[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) wt[i] = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[i].x - M);
  if (tid < own) s_w[tid] = wt[0];
  if (tid < pieces) s_w[own + tid] = wt[1];
  const float lsum = wave_all(wt[0] * ml[0].y + wt[1] * ml[1].y, Add());
  if (lane == 0) s_red[4 + wave] = lsum;
  __syncthreads();
  const float L = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int c, const float4& x) {
    const float w = s_w[c];
    a.x += w * x.x;
    a.y += w * x.y;
    a.z += w * x.z;
    a.w += w * x.w;
  };
#pragma unroll
  for (int i = 0; i < kMergeAhead; ++i)
    if (g + 8 * i < all) add(g + 8 * i, ahead[i]);
#pragma unroll 4
  for (int c = g + 8 * kMergeAhead; c < all; c += 8) add(c, *part(c));
  s_part[g][q] = a;
  __syncthreads();
  if (tid < kD) {
    const float* sums = reinterpret_cast<const float*>(s_part) + tid;
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc += sums[i * kD];
    p.out[row * kD + tid] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(acc / L));   // no key: 0 / 0
    if (tid == 0) p.lse[row] = M == -INFINITY && L == L ? -INFINITY : M + log2f(L);
  }
}

constexpr int kTarget = 2;         // workgroups per CU
constexpr int kLineLeast = 8;      // of the target, the part that the line gets at least
// Own rows are read past the 256 MB memory-side cache where it cannot hold caches and
// prefixes: B64 of 1024 rows behind 8192 54.4 -> 51.7 us.  Smaller ones may still be there
// from the last call: B40 of 777 rows 30.5 us, streamed 32.6.
constexpr int64_t kStreamBytes = int64_t{256} << 20;
// Prefixes too, from a size on that other layers' rows push out before the next step, where one
// tile takes all sequences: one of 30720 rows, 8 KV heads, B20 39.9 -> 34.8 us, B1 of 32768 35.4 ->
// 32.8.  Tiles that share a prefix find it in the caches: B64 Hq64 behind 32768 136, streamed 141.
constexpr int64_t kStreamPrefixBytes = int64_t{96} << 20;

int shared_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    return 256;
  return n;
}

struct SharedLayout {
  int64_t slots, pieces, tile_seqs, tile_rows, target, least;
  int64_t off_ml, off_plan, off_place, off_tile_o, off_tile_ml, bytes;
};

// Bounds on what the device plans: tiles are at most one per sequence, and one begun
// per group and one per tile_seqs sequences; pieces the target's shares and one more
// for each (tile, KV head).
bool shared_layout(int64_t batch, int64_t cache_len, int64_t prefixes, int64_t prefix_len, int64_t hq, int64_t hkv,
                   SharedLayout& L) {
  if (batch < 1 || batch > SWATTN_SHARED_MAX_SEQS || prefixes < 1 || prefixes > SWATTN_SHARED_MAX_PREFIXES) return false;
  if (cache_len < 1 || prefix_len < 1 || cache_len > INT32_MAX || prefix_len > INT32_MAX) return false;
  if (hq < 1 || hkv < 1 || hkv > 65535 || hq % hkv != 0 || hq / hkv > kMaxG) return false;
  const int64_t group = hq / hkv;
  L.tile_seqs = kTileRows / group;
  const int64_t by_group = 2 * prefixes + batch / L.tile_seqs, tiles = by_group < batch ? by_group : batch;
  // The line takes kPairPad positions per pair beside its keys; pieces are whole key tiles.
  if (batch * hkv * (cache_len + kPairPad) > INT32_MAX || tiles * hkv * (prefix_len + kTileKeys) > INT32_MAX) return false;
  L.tile_rows = (batch < L.tile_seqs ? batch : L.tile_seqs) * group;
  L.target = int64_t{kTarget} * shared_cus();
  L.least = (L.target + kLineLeast - 1) / kLineLeast;
  L.slots = L.target + L.least + batch * hkv;
  L.pieces = L.target + tiles * hkv;
  // A launch takes fewer than 2^32 threads: the merge 256 per output row (pieces are fewer, a
  // pair's start and its keys being positions of the line).
  if (batch * hq >= int64_t{1} << 24) return false;
  auto al = [](int64_t x) { return (x + 255) & ~int64_t{255}; };
  int64_t o = al(L.slots * group * kD * 4);
  L.off_ml = o;       o = al(o + L.slots * group * 2 * 4);
  L.off_plan = o;     o = al(o + (1 + batch) * 16);
  L.off_place = o;    o = al(o + batch * 16);
  L.off_tile_o = o;   o = al(o + L.pieces * L.tile_rows * kD * 4);
  L.off_tile_ml = o;  o = al(o + L.pieces * L.tile_rows * 2 * 4);
  L.bytes = o;
  return true;
}

// What the plan goes by of a call's sizes.
void plan_sizes(SharedParams& p, const SharedLayout& L, int32_t batch, int64_t cache_len, int32_t prefixes, int64_t prefix_len,
                int32_t heads_q, int32_t heads_kv, int32_t window) {
  p.cache_len = static_cast<int>(cache_len);
  p.batch = batch;
  p.hq = heads_q;
  p.hkv = heads_kv;
  p.group = heads_q / heads_kv;
  p.window = window;
  p.target = static_cast<uint32_t>(L.target);
  p.target_inv = static_cast<uint32_t>(((int64_t{1} << 32) + L.target - 1) / L.target);
  p.pad = kPairPad;
  p.prefixes = prefixes;
  p.prefix_len = static_cast<int>(prefix_len);
  p.tile_seqs = static_cast<int>(L.tile_seqs);
  p.tile_inv = static_cast<uint32_t>((1u << 20) / L.tile_seqs + 1);
  p.tile_rows = static_cast<int>(L.tile_rows);
  p.least = static_cast<uint32_t>(L.least);
}

}  // namespace
}  // namespace swattn

using namespace swattn;

extern "C" {

size_t swattn_shared_decode_workspace_bytes(int32_t batch, int64_t cache_len, int32_t prefixes, int64_t prefix_len,
                                            int32_t heads_q, int32_t heads_kv) {
  SharedLayout L;
  return shared_layout(batch, cache_len, prefixes, prefix_len, heads_q, heads_kv, L) ? static_cast<size_t>(L.bytes) : 0;
}

int swattn_shared_decode_fwd(const void* q, const void* k_prefix, const void* v_prefix, const int32_t* prefix_lens,
                             const int32_t* prefix_ids, const void* k_cache, const void* v_cache,
                             const int32_t* cache_lens, const uint8_t* full, void* out, float* lse, int32_t batch,
                             int64_t cache_len, int32_t prefixes, int64_t prefix_len, int32_t heads_q,
                             int32_t heads_kv, int32_t head_dim, int32_t window, float scale_log2, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* name = "swattn_shared_decode_fwd";
  const std::string n(name);
  if (head_dim != kD) return invalid(n + ": head_dim must be 128");
  if (batch < 1 || cache_len < 1 || prefixes < 1 || prefix_len < 1 || heads_q < 1 || heads_kv < 1)
    return invalid(n + ": bad shape");
  if (heads_q % heads_kv) return invalid(n + ": heads_q must be a multiple of heads_kv");
  if (heads_q / heads_kv > kMaxG) return invalid(n + ": heads_q / heads_kv must be at most 8");
  if (window <= 0) return invalid(n + ": window must be positive");
  if (!isfinite(scale_log2)) return invalid(n + ": scale_log2 must be finite");
  SharedLayout L;
  if (!shared_layout(batch, cache_len, prefixes, prefix_len, heads_q, heads_kv, L))
    return invalid(n + ": batch, prefixes, heads_kv or the lengths too large");
  if (q == nullptr || k_prefix == nullptr || v_prefix == nullptr || prefix_lens == nullptr || prefix_ids == nullptr ||
      k_cache == nullptr || v_cache == nullptr || cache_lens == nullptr || full == nullptr || out == nullptr || lse == nullptr)
    return invalid(n + ": null pointer");
  if (!aligned16(q) || !aligned16(k_prefix) || !aligned16(v_prefix) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return invalid(n + ": q, the prefixes, the caches and out must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(L.bytes)) {
    set_error(n + ": workspace smaller than swattn_shared_decode_workspace_bytes()");
    return SWATTN_EWORKSPACE;
  }
  if (!aligned256(workspace)) return invalid(n + ": workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  SharedParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k_cache);
  p.v = static_cast<const uint16_t*>(v_cache);
  p.c = scale_log2;
  p.lens = cache_lens;
  p.full = full;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + L.off_ml);
  p.plan = reinterpret_cast<uint4*>(ws + L.off_plan);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  plan_sizes(p, L, batch, cache_len, prefixes, prefix_len, heads_q, heads_kv, window);
  p.prefix_k = static_cast<const uint16_t*>(k_prefix);
  p.prefix_v = static_cast<const uint16_t*>(v_prefix);
  p.prefix_lens = prefix_lens;
  p.prefix_ids = prefix_ids;
  p.tile_o = reinterpret_cast<float*>(ws + L.off_tile_o);
  p.tile_ml = reinterpret_cast<float*>(ws + L.off_tile_ml);
  p.place = reinterpret_cast<int4*>(ws + L.off_place);
  p.stream_prefix = batch <= L.tile_seqs && prefixes * prefix_len * heads_kv * (4 * kD) >= kStreamPrefixBytes;
  const hipStream_t st = as_stream(stream);
  const dim3 grid(static_cast<uint32_t>(L.pieces + L.least));
  const bool stream_past = (batch * cache_len + prefixes * prefix_len) * heads_kv * (4 * kD) >= kStreamBytes;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p); };
  if (batch > 256 || prefixes > 256) {
    if (stream_past)
      launch(shared_split_kernel<kMostPer, true>);
    else
      launch(shared_split_kernel<kMostPer, false>);
  } else if (stream_past) {
    launch(shared_split_kernel<1, true>);
  } else {
    launch(shared_split_kernel<1, false>);
  }
  hipLaunchKernelGGL(shared_merge_kernel, dim3(static_cast<uint32_t>(p.group), static_cast<uint32_t>(heads_kv), static_cast<uint32_t>(batch)),
                     dim3(256), 0, st, p);
  return launch_status(name);
}

int swattn_shared_plan(const int32_t* prefix_lens, const int32_t* prefix_ids, const int32_t* cache_lens, const uint8_t* full,
                       int32_t batch, int64_t cache_len, int32_t prefixes, int64_t prefix_len, int32_t heads_q,
                       int32_t heads_kv, int32_t window, int64_t* totals, int32_t* pieces, int64_t max_pieces, int64_t* own) {
  SharedLayout L;
  if (window <= 0 || !shared_layout(batch, cache_len, prefixes, prefix_len, heads_q, heads_kv, L))
    return invalid("swattn_shared_plan: shapes that the decode refuses");
  SharedParams p{};
  plan_sizes(p, L, batch, cache_len, prefixes, prefix_len, heads_q, heads_kv, window);
  auto clamped = [](int32_t x, int most) { return x < 0 ? 0 : x > most ? most : x; };
  struct Group {
    uint32_t seqs, first;
  };
  Group groups[2 * SWATTN_SHARED_MAX_PREFIXES];
  uint32_t keys[SWATTN_SHARED_MAX_SEQS];
  for (int i = 0; i < 2 * prefixes; ++i) groups[i] = Group{0u, UINT32_MAX};
  uint32_t all_keys = 0, all_cnt = 0;
  for (int b = 0; b < batch; ++b) {
    const int len = clamped(cache_lens[b], p.cache_len), id = prefix_ids[b];
    keys[b] = full[b] ? len : len < window ? len : window;
    all_keys += keys[b];
    all_cnt += keys[b] > 0 ? 1 : 0;
    if (id < 0 || id >= prefixes) continue;
    const int rows = clamped(prefix_lens[id], p.prefix_len), start = prefix_start(full[b] != 0, rows, len, window);
    if (start >= rows) continue;
    Group& g = groups[2 * id + (full[b] ? 0 : 1)];
    ++g.seqs;
    if (static_cast<uint32_t>(start) < g.first) g.first = start;
  }
  auto keys_of = [&](int i) { return static_cast<uint32_t>(clamped(prefix_lens[i / 2], p.prefix_len)) - groups[i].first; };
  uint32_t positions = 0;
  for (int i = 0; i < 2 * prefixes; ++i)
    if (groups[i].seqs > 0) positions += tiles_of(groups[i].seqs, p.tile_seqs, p.tile_inv) * keys_of(i);
  const uint32_t line = (all_keys + all_cnt * p.pad) * p.hkv;
  const uint32_t length = piece_length(line, positions, p.hkv, p.target_inv, p.prefix_len);
  uint32_t base = 0;
  for (int i = 0; i < 2 * prefixes; ++i) {
    if (groups[i].seqs == 0) continue;
    const uint32_t tiles = tiles_of(groups[i].seqs, p.tile_seqs, p.tile_inv), n = keys_of(i);
    const Cut cut = cut_keys(n, length);
    const uint32_t here = tiles * p.hkv * cut.parts;
    for (uint32_t at = 0; at < here && base + at < max_pieces; ++at) {
      const PieceOf x = piece_of(at, here, tiles, cut.parts);
      const uint32_t from = x.part * cut.length, to = from + cut.length < n ? from + cut.length : n;
      const uint32_t row[8] = {static_cast<uint32_t>(i / 2), static_cast<uint32_t>(i & 1), x.tile, x.kvh, groups[i].first + from,
                               groups[i].first + to, base + (x.tile * p.hkv + x.kvh) * cut.parts + x.part, cut.parts};
      for (int j = 0; j < 8; ++j) pieces[8 * (static_cast<int64_t>(base) + at) + j] = static_cast<int32_t>(row[j]);
    }
    base += here;
  }
  p.target = line_target(p.target, base, p.least);
  Line<uint32_t> S = plan_line<uint32_t>(p, all_keys * p.hkv, all_cnt * p.hkv);
  uint32_t total = 0, rank = 0;
  int64_t slots = 0;
  const uint32_t inv = UINT32_MAX / S.share;
  for (int b = 0; b < batch; ++b) {
    const uint32_t len = S.length(keys[b], p.pad);
    for (int kvh = 0; kvh < p.hkv; ++kvh) {
      int64_t* to = own + 4 * (static_cast<int64_t>(b) * p.hkv + kvh);
      const uint32_t wg0 = share_of(total, S.share, inv);
      to[0] = total;
      to[1] = keys[b];
      to[2] = static_cast<int64_t>(wg0) + static_cast<int64_t>(rank) * p.hkv + kvh;
      to[3] = keys[b] > 0 ? share_of(total + keys[b] - 1, S.share, inv) - wg0 + 1 : 0;
      if (to[3] > 0 && to[2] + to[3] > slots) slots = to[2] + to[3];
      total += len;
    }
    rank += keys[b] > 0 ? 1 : 0;
  }
  const int64_t out[8] = {base, L.pieces, (static_cast<int64_t>(total) + S.share - 1) / S.share, slots, L.slots, L.pieces + L.least,
                          S.share, total};
  for (int i = 0; i < 8; ++i) totals[i] = out[i];
  return SWATTN_OK;
}

}  // extern "C"
