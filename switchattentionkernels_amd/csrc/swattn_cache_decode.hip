// Routed GQA decode over an 8-bit KV cache for gfx950 (include/swattn_cache.h):
// the rule of swattn_decode.hip, with keys and values code * scale, one scale
// per block of tokens and KV head, and on request the sum over a KV head's query
// heads of each key's softmax weight.  No counterpart in the reference.
//
//   s_j = c ks_j (q . kc_j),  p_j = 2^(s_j - m),  l = sum p_j,
//   o = sum (p_j vs_j) vc_j / l,  LSE = m + log2 l,  w_j += sum_heads 2^(s_j - LSE)
// kc, vc codes, ks, vs their scales: a scale multiplies a score or a weight, not
// 128 values.
//
// HBM-bound: 256 bytes and two scales per key and KV head.  The routed keys of
// all pairs form one line that the workgroups share out (decode_line.h).  With
// half the bytes per key of a bf16 cache the vector ALUs no longer keep up with
// a dot product per head (8 heads: 2048 multiply-adds and 256 conversions per
// key, about twice the time the key takes to arrive); the products run on the
// matrix cores, codes converted to bf16 (exact for both codes):
// * S^T [16 keys x 16 columns] = K Q^T, v_mfma_f32_16x16x32_bf16.  Lane (r, g) =
//   (lane % 16, lane / 16) holds key r of the tile, bytes 16 g .. +15 of both
//   64-byte halves of its row: the A operand needs no exchange between lanes.
// * O^T [16 dims x 16 columns] += V^T P^T for eight tiles of dims, 32 keys at
//   once.  Lane (c, g) holds dims 8 c .. +7 of keys 4 g .. +3 of both key tiles;
//   tile n takes dim 8 c + n of each, so that S^T's accumulator layout (column
//   lane % 16, keys 4 g .. +3) is P's operand layout, and V is transposed
//   inside a lane.
// * p vs enters the product with V as three bf16 numbers, its value, what that leaves
//   and what both leave: 24 bits, as in fp32.  A group has at most 8 heads and the
//   tiles have 16 columns: columns 8-15 repeat the heads and take the second where
//   columns 0-7 take the first; the third needs a product of its own.  Without it (17
//   bits) 206 of 131072 outputs of 32768 keys were rounded to the wrong side, 29 with
//   it and 122 by fp32 sums; it costs 0.3 us of 157.4 there, 1.5 of 72.4 at B64.
//
// Measured, Hkv 8, as a large copy's 5.2 TB/s goes: B16 L16384-32768 Hq64 int8 all
// full 158 us, 5.1 TB/s of codes and scales; B64 L4096-8192 Hq32 e4m3 p_full
// 0.25 72-74 us, of which the merge and its launch are about 8; B1 L4096 Hq32 11.3 us, bound
// by dependent latencies (plan, first keys, combine, merge) and, at that length, by
// the host's calls.  Two workgroups per CU with loads three steps ahead: 12.8 us
// (B1), 77 (B64); four with one step ahead 13 and 85.  Joining the pieces in the same
// launch, the last workgroup of a pair waiting for the others' tags, took half
// as long again (B64 104 us): every release writes an L2 back.

#include <limits.h>
#include <math.h>

#include <atomic>
#include <string>

#include "cache_code.h"
#include "decode_line.h"

namespace swattn {
namespace {

using namespace code;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;            // waves per workgroup
constexpr int kMaxG = 8;
constexpr int kStep = 32;            // keys a wave takes at once
constexpr int kAhead = 1;            // steps a wave's loads run ahead
constexpr uint32_t kPairPad = 192;   // a pair's start, in keys

struct CacheDecodeParams : DecodeCommon {
  static constexpr uint32_t kMinShare = 128;     // line positions per workgroup, at least
  static constexpr uint32_t kLongShare = 4096;   // shares from this length on are halved
  static constexpr uint32_t kAlignSlack = 160;
  static constexpr bool kKeepNan = true;         // a block that took a NaN shows in every row that attends it
  const uint16_t* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scales;
  const float* v_scales;
  float* scores;      // [B][Hq][score_len] exp2-domain scores of the attended keys, or null
  float* weights;     // [B][Hkv][cache_len], or null
  int64_t score_len;
  int nblk, block_log;
  int weight_wgs;     // workgroups that add weights, per (sequence, KV head)
  float c;            // sm_scale * log2(e)
};

// Two codes (bytes 2 i, 2 i + 1 of w) as a bf16 pair.
template <int kCode, bool kHigh>
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w) {
  if constexpr (kCode == kE4m3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
  } else {
    const float a = static_cast<float>(static_cast<int8_t>(w >> (kHigh ? 16 : 0)));
    const float b = static_cast<float>(static_cast<int8_t>(w >> (kHigh ? 24 : 8)));
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
}
template <int kCode>
__device__ __forceinline__ bf16x8 eight_bf16(uint32_t lo, uint32_t hi) {
  const u32x4 u = {pair_bf16<kCode, false>(lo), pair_bf16<kCode, true>(lo), pair_bf16<kCode, false>(hi),
                   pair_bf16<kCode, true>(hi)};
  return __builtin_bit_cast(bf16x8, u);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const bf16x2 x = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, x);
}

// Caches that the 256 MB memory-side cache cannot hold are streamed past it: B64 of
// 8192 rows, 8 KV heads 73.4 -> 70.7 us, B16 of 32768 169 -> 163.  Smaller ones may
// still be there from the last call: B24 of 2999 29.7 us, streamed 35.6; B8 of 4096
// 17.5 and 18.9.
constexpr int64_t kStreamBytes = int64_t{256} << 20;

// One step's data: 32 keys of K and V and the scales of both key tiles.
struct Step {
  uint4 k[2][2];   // [key tile][64-byte half of the row]
  uint2 v[8];      // keys 4 g + t of tile t / 4
  float scale;     // lane % 4: K tile 0, K tile 1, V tile 0, V tile 1
};

// One workgroup per share of the line, as decode_split_kernel.  Wave w takes the
// 32-key steps w, w + 4, ... of a piece, which begin at multiples of 32 of the
// sequence; rows outside the piece are read as its nearest row and masked.
template <int kCode, bool kInline, bool kScores, bool kStream>
__global__ __launch_bounds__(256, 3) void cache_split_kernel(const CacheDecodeParams p) {
  __shared__ float s_m[kWaves][kMaxG], s_l[kWaves][kMaxG];
  __shared__ float s_acc[kWaves][kMaxG][kD];
  __shared__ SeqEntry s_ent[kInline ? kInlineSeqs : 1];
  SplitStart st;
  if constexpr (kInline) {
    if (!plan_inline(p, s_ent, st)) return;
  } else {
    if (!plan_listed(p, st)) return;
  }
  auto uniform = [](uint32_t x) { return static_cast<int>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); };
  int r = uniform(st.r), kvh = uniform(st.kvh);
  uint32_t key = uniform(st.key);
  uint32_t left = uniform(st.take);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int G = p.group;
  const int head = c & 7;          // of the group; columns 8-15 repeat them
  const bool error_col = c >= 8;
  const int64_t stride = static_cast<int64_t>(p.hkv) * kD;   // bytes per cache row
  for (;;) {
    SeqEntry e;
    if constexpr (kInline) {
      e = s_ent[r];
    } else {
      e.b = p.list[r];
      key_range(p, e.b, e.lo, e.n);
      e.len = p.plan[1 + e.b].w;
    }
    const int b = uniform(e.b);
    const uint32_t n = uniform(e.n), len = uniform(e.len);
    const uint32_t took = min(left, len - key);
    left -= took;
    if (key < n) {   // else this share starts in the pair's padding
      const int64_t slot = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(r) * p.hkv + kvh;
      const int k0 = uniform(e.lo) + static_cast<int>(key), k1 = k0 + static_cast<int>(min(took, n - key));
      const int64_t pair = static_cast<int64_t>(b) * p.hkv + kvh;
      // Q^T operands: dims 64 j + 16 g + 8 i .. +7 of column c's head.
      bf16x8 q[2][2];
      const uint16_t* qp = p.q + (static_cast<int64_t>(b) * p.hq + kvh * G + min(head, G - 1)) * kD + 16 * g;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u32x4 u = *reinterpret_cast<const u32x4*>(qp + 64 * j + 8 * i);
          if (head >= G) u = u32x4{0, 0, 0, 0};
          q[j][i] = __builtin_bit_cast(bf16x8, u);
        }
      const uint8_t* kb = p.k + static_cast<int64_t>(b) * p.cache_len * stride + kvh * kD + 16 * g;
      const uint8_t* vb = p.v + static_cast<int64_t>(b) * p.cache_len * stride + kvh * kD + 8 * c;
      const float* sb = (lane & 2 ? p.v_scales : p.k_scales) + pair * p.nblk;
      const int base = k0 & ~(kStep - 1);
      const int steps = (k1 - base + kStep - 1) / kStep;   // of the piece; this wave's: wave, wave + 4, ...
      auto load = [&](int i, Step& s) {
        const int kk = base + kStep * i;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int row = min(max(kk + 16 * t + c, k0), k1 - 1);
          const uint8_t* at = kb + row * stride;
          s.k[t][0] = load_bytes<kStream, u32x4, uint4>(at);
          s.k[t][1] = load_bytes<kStream, u32x4, uint4>(at + 64);
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const int row = min(max(kk + 16 * (t >> 2) + 4 * g + (t & 3), k0), k1 - 1);
          s.v[t] = load_bytes<kStream, uint64_t, uint2>(vb + row * stride);
        }
        // Of a tile without a row of the piece: the scale of the nearest block, not
        // a block that may hold no valid row.
        s.scale = sb[min(max(kk + 16 * (lane & 1), k0), k1 - 1) >> p.block_log];
      };
      Step ring[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) load(wave + kWaves * j, ring[j]);
      float m = -INFINITY, l = 0.f;   // column c's maximum, and this lane's share of its sum
      f32x4 acc[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int i0 = wave; i0 < steps; i0 += kWaves * kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int i = i0 + kWaves * j;
          if (i >= steps) break;
          Step& d = ring[j];
          const int kk = base + kStep * i;
          const float ds = d.scale;
          auto scale_of = [&](int x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ds), x)); };
          const float ks[2] = {scale_of(0) * p.c, scale_of(1) * p.c}, vs[2] = {scale_of(2), scale_of(3)};
          f32x4 s[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<kCode>(d.k[t][u].x, d.k[t][u].y), q[u][0], s[t], 0, 0, 0);
              s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<kCode>(d.k[t][u].z, d.k[t][u].w), q[u][1], s[t], 0, 0, 0);
            }
            s[t] *= ks[t];
          }
          // Keys of the piece: kk + 16 t + 4 g + e.
          const bool whole = kk >= k0 && kk + kStep <= k1;   // uniform
          bool live[2][4];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int at = kk + 16 * t + 4 * g + x;
              live[t][x] = whole || (at >= k0 && at < k1);
              if (!live[t][x]) s[t][x] = -INFINITY;
            }
          if constexpr (kScores) {
            if (c < G) {
              float* sp = p.scores + (static_cast<int64_t>(b) * p.hq + kvh * G + c) * p.score_len + kk + 4 * g;
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                if (whole) {
                  *reinterpret_cast<f32x4*>(sp + 16 * t) = s[t];
                } else {
#pragma unroll
                  for (int x = 0; x < 4; ++x)
                    if (live[t][x]) sp[16 * t + x] = s[t][x];
                }
              }
            }
          }
          float top = s[0][0];
#pragma unroll
          for (int x = 1; x < 8; ++x) top = fmaxf(top, s[x >> 2][x & 3]);
          if (__builtin_amdgcn_ballot_w64(top - m > 8.0f)) {   // rare: move the maxima, rescale
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = top - m > 8.0f ? top : m;
            const float a = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= a;
#pragma unroll
            for (int t = 0; t < 8; ++t) acc[t] *= a;
          }
          // Only scores of -inf so far (products past fp32's range): they weigh nothing.
          const float from = m == -INFINITY ? 0.f : m;
          u32x4 pk, pk2;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 4; x += 2) {
              float y[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float pr = live[t][x + i] ? __builtin_amdgcn_exp2f(s[t][x + i] - from) : 0.f;
                l += pr;
                y[i] = pr * vs[t];
              }
              const uint32_t high = pack2(y[0], y[1]);   // the differences are exact
              y[0] -= __uint_as_float(high << 16);
              y[1] -= __uint_as_float(high & 0xffff0000u);
              const uint32_t mid = pack2(y[0], y[1]);
              y[0] -= __uint_as_float(mid << 16);
              y[1] -= __uint_as_float(mid & 0xffff0000u);
              pk[2 * t + x / 2] = error_col ? mid : high;
              pk2[2 * t + x / 2] = error_col ? 0u : pack2(y[0], y[1]);
            }
          const bf16x8 pb = __builtin_bit_cast(bf16x8, pk), pb2 = __builtin_bit_cast(bf16x8, pk2);
          // V^T operands of dims 2 d, 2 d + 1 of this lane's eight: pairs of keys.
#pragma unroll
          for (int d2 = 0; d2 < 4; ++d2) {
            u32x4 a0, a1;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint32_t w0 = d2 & 2 ? d.v[2 * t].y : d.v[2 * t].x, w1 = d2 & 2 ? d.v[2 * t + 1].y : d.v[2 * t + 1].x;
              const uint32_t x0 = d2 & 1 ? pair_bf16<kCode, true>(w0) : pair_bf16<kCode, false>(w0);
              const uint32_t x1 = d2 & 1 ? pair_bf16<kCode, true>(w1) : pair_bf16<kCode, false>(w1);
              a0[t] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
              a1[t] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
            }
            acc[2 * d2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), pb, acc[2 * d2], 0, 0, 0);
            acc[2 * d2 + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), pb, acc[2 * d2 + 1], 0, 0, 0);
            acc[2 * d2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), pb2, acc[2 * d2], 0, 0, 0);
            acc[2 * d2 + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), pb2, acc[2 * d2 + 1], 0, 0, 0);
          }
          load(i + kWaves * kAhead, d);   // refill the slot; past the end: clamped, never used
        }
      }
      // This wave's partial: column c's sum over its four lanes, and O^T with its
      // error columns (by shuffles, as in the maxima's move above: lane moves there cost
      // the loop its register allocation, B16 158 -> 161 us).  acc[t][x]: dim 8 (4 g + x) + t of column c.
      l = with_lane32(with_lane16(l, Add()), Add());
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[t][x] += __shfl_xor(acc[t][x], 8);
      if (c < G) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int t = 0; t < 8; t += 4)
            *reinterpret_cast<f32x4*>(&s_acc[wave][c][8 * (4 * g + x) + t]) =
                f32x4{acc[t][x], acc[t + 1][x], acc[t + 2][x], acc[t + 3][x]};
        if (g == 0) {
          s_m[wave][c] = m;
          s_l[wave][c] = l;
        }
      }
      __syncthreads();
      // Combine the waves: one partial (unnormalised acc, max, sum) per head.
      float* po = p.part_o + slot * G * kD;
      float* pml = p.part_ml + slot * G * 2;
      for (int i = tid; i < G * kD; i += 256) {
        const int h = i / kD, d = i - h * kD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_m[w][h]);
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          if (s_l[w][h] != 0.f) a += exp2f(s_m[w][h] - mm) * s_acc[w][h][d];
        po[i] = a;
      }
      if (tid < G) {
        float mm = -INFINITY, lh = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_m[w][tid]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          if (s_l[w][tid] != 0.f) lh += exp2f(s_m[w][tid] - mm) * s_l[w][tid];
        pml[2 * tid] = mm;
        pml[2 * tid + 1] = lh;
      }
    }
    // The rest of the share continues at the start of the next pair.
    if (left == 0u) return;
    key = 0;
    if (++kvh == p.hkv) {
      kvh = 0;
      ++r;
    }
    __syncthreads();   // the next piece's combine writes the same LDS
  }
}

// Workgroups below batch * hq merge an output row each; the rest add the weights
// of kWeightKeys keys of one (sequence, KV head) each, a thread per key, from the
// scores and the pair's LSEs, which they compute from the partials as the merge
// does.
constexpr int kWeightKeys = 256;
__global__ __launch_bounds__(256) void cache_merge_kernel(const CacheDecodeParams p) {
  const int64_t rows = static_cast<int64_t>(p.batch) * p.hq;
  if (blockIdx.x < rows) {
    merge_row(p, blockIdx.x);
    return;
  }
  __shared__ float s_lse[kMaxG];
  const int64_t x = blockIdx.x - rows;
  const int64_t pair = x / p.weight_wgs;
  const int b = static_cast<int>(pair / p.hkv), kvh = static_cast<int>(pair - static_cast<int64_t>(b) * p.hkv);
  int lo, n;
  key_range(p, b, lo, n);
  // Chunks at multiples of kWeightKeys of the sequence, from the one with lo on.
  const int64_t first = static_cast<int64_t>(lo / kWeightKeys + (x - pair * p.weight_wgs)) * kWeightKeys;
  if (first >= lo + static_cast<int64_t>(n)) return;   // uniform
  const SeqPlace seq = seq_place(p.plan[1 + b]);
  const uint32_t share = p.plan[0].x;
  const uint64_t off = seq.off + static_cast<uint64_t>(kvh) * seq.len;
  const uint32_t wg0 = quotient(off, share);
  const int nch = static_cast<int>(quotient(off + seq.n - 1, share) - wg0) + 1;
  const int64_t slot0 = static_cast<int64_t>(wg0) + static_cast<int64_t>(seq.rank) * p.hkv + kvh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, G = p.group;
  const int64_t j = first + threadIdx.x;
  const bool live = j >= lo && j < lo + static_cast<int64_t>(n);
  const float* sc = p.scores + (static_cast<int64_t>(b) * p.hq + kvh * G) * p.score_len + j;
  float score[kMaxG];
#pragma unroll
  for (int h = 0; h < kMaxG; ++h) score[h] = live && h < G ? sc[h * p.score_len] : -INFINITY;
  float* w = p.weights + pair * p.cache_len + j;
  const float before = live ? *w : 0.f;
  for (int h = wave; h < G; h += 4) {
    float mx = -INFINITY, sum = 0.f;
    float2 ml[kMaxSplitsDev / 64];
#pragma unroll
    for (int i = 0; i < kMaxSplitsDev / 64; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      const int s = lane + 64 * i;
      if (s < nch) ml[i] = *reinterpret_cast<const float2*>(p.part_ml + ((slot0 + s) * G + h) * 2);
      mx = fmaxf(mx, ml[i].x);
    }
    mx = wave_all(mx, Max());
#pragma unroll
    for (int i = 0; i < kMaxSplitsDev / 64; ++i)
      if (ml[i].y != 0.f) sum += __builtin_amdgcn_exp2f(ml[i].x - mx) * ml[i].y;
    sum = wave_all(sum, Add());
    if (lane == 0) s_lse[h] = mx + log2f(sum);
  }
  __syncthreads();
  if (!live) return;
  float sum = 0.f;
#pragma unroll
  for (int h = 0; h < kMaxG; ++h)
    if (h < G) sum += __builtin_amdgcn_exp2f(score[h] - s_lse[h]);
  *w = before + sum;
}

// Workgroups that the line is shared out over: three per CU, as many as are
// resident at once; the workspace holds six per CU plus one per pair partials.
constexpr int kSplitTarget = 3;
constexpr int kSplitRoom = 6;
static_assert(2 * kSplitTarget <= kSplitRoom, "every share has its partial");

// Compute units of the current device, looked up once per device.
int cu_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 256;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

struct Layout {
  int64_t slots, score_len, off_ml, off_list, off_plan, off_scores, bytes;
};

Layout layout(int64_t batch, int64_t cache_len, int64_t heads_q, int64_t heads_kv, bool with_weights, int cus) {
  Layout L{};
  L.slots = static_cast<int64_t>(kSplitRoom) * cus + batch * heads_kv;
  L.score_len = (cache_len + kStep - 1) / kStep * kStep;
  const int64_t group = heads_q / heads_kv;
  auto al = [](int64_t x) { return (x + 255) & ~static_cast<int64_t>(255); };
  int64_t o = al(L.slots * group * kD * 4);   // part_o
  L.off_ml = o;      o = al(o + L.slots * group * 2 * 4);
  L.off_list = o;    o = al(o + batch * 4);
  L.off_plan = o;    o = al(o + (1 + batch) * 16);
  L.off_scores = o;  if (with_weights) o = al(o + batch * heads_q * L.score_len * 4);
  L.bytes = o;
  return L;
}

template <int kCode, bool kInline, bool kScores>
void launch_split(bool streamed, dim3 grid, hipStream_t st, const CacheDecodeParams& p) {
  if (streamed)
    hipLaunchKernelGGL((cache_split_kernel<kCode, kInline, kScores, true>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((cache_split_kernel<kCode, kInline, kScores, false>), grid, dim3(256), 0, st, p);
}
template <int kCode>
void launch_split(bool inline_plan, bool streamed, dim3 grid, hipStream_t st, const CacheDecodeParams& p) {
  if (inline_plan)
    p.scores != nullptr ? launch_split<kCode, true, true>(streamed, grid, st, p)
                        : launch_split<kCode, true, false>(streamed, grid, st, p);
  else
    p.scores != nullptr ? launch_split<kCode, false, true>(streamed, grid, st, p)
                        : launch_split<kCode, false, false>(streamed, grid, st, p);
}

}  // namespace
}  // namespace swattn

using namespace swattn;

extern "C" {

size_t swattn_cache_decode_workspace_bytes(int32_t batch, int64_t cache_len, int32_t heads_q,
                                           int32_t heads_kv, int32_t with_weights) {
  if (batch < 1 || cache_len < 1 || cache_len > INT32_MAX || heads_q < 1 || heads_kv < 1 || heads_q % heads_kv)
    return 0;
  return static_cast<size_t>(layout(batch, cache_len, heads_q, heads_kv, with_weights != 0, cu_count()).bytes);
}

int swattn_cache_decode_fwd(const void* q, const void* k, const void* v, const float* k_scales,
                            const float* v_scales, const int32_t* cache_lens, const uint8_t* full,
                            void* out, float* lse, float* key_weights, int32_t batch,
                            int64_t cache_len, int32_t heads_q, int32_t heads_kv,
                            int32_t head_dim, int32_t window, int32_t block, int32_t codes,
                            float scale_log2, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const std::string n("swattn_cache_decode_fwd");
  if (head_dim != kD) return invalid(n + ": head_dim must be 128");
  if (batch < 1 || cache_len < 1 || heads_q < 1 || heads_kv < 1) return invalid(n + ": bad shape");
  if (heads_q % heads_kv) return invalid(n + ": heads_q must be a multiple of heads_kv");
  if (heads_q / heads_kv > kMaxG) return invalid(n + ": heads_q / heads_kv must be at most 8");
  if (window <= 0) return invalid(n + ": window must be positive");
  if (batch > 65535 || heads_kv > 65535 || cache_len > INT32_MAX - 256 ||
      static_cast<int64_t>(batch) * heads_q > INT32_MAX)
    return invalid(n + ": batch, heads_kv or cache_len too large");
  if (!block_ok(block)) return invalid(n + ": block must be 16, 32, 64 or 128");
  if (codes != kE4m3 && codes != kInt8) return invalid(n + ": unknown code");
  if (q == nullptr || k == nullptr || v == nullptr || k_scales == nullptr || v_scales == nullptr ||
      cache_lens == nullptr || full == nullptr || out == nullptr || lse == nullptr)
    return invalid(n + ": null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return invalid(n + ": q, k, v and out must be 16-byte aligned");
  const int cus = cu_count();
  const Layout L = layout(batch, cache_len, heads_q, heads_kv, key_weights != nullptr, cus);
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(L.bytes)) {
    set_error(n + ": workspace smaller than swattn_cache_decode_workspace_bytes()");
    return SWATTN_EWORKSPACE;
  }
  if (!aligned256(workspace)) return invalid(n + ": workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  const int64_t pairs = static_cast<int64_t>(batch) * heads_kv, rows = pairs * cache_len;
  if (L.slots > INT32_MAX) return invalid(n + ": too many work items");
  CacheDecodeParams p{};
  p.target = kSplitTarget * cus;
  if (rows / p.target >= (int64_t{1} << 30)) return invalid(n + ": the K cache is larger than the address space");
  p.lens = cache_lens;
  p.full = full;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + L.off_ml);
  p.list = reinterpret_cast<int32_t*>(ws + L.off_list);
  p.plan = reinterpret_cast<uint4*>(ws + L.off_plan);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.cache_len = static_cast<int>(cache_len);
  p.batch = batch;
  p.hq = heads_q;
  p.hkv = heads_kv;
  p.group = heads_q / heads_kv;
  p.window = window;
  p.pad = pairs < (int64_t{1} << 30) / kPairPad ? kPairPad : 0;
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint8_t*>(k);
  p.v = static_cast<const uint8_t*>(v);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.scores = key_weights != nullptr ? reinterpret_cast<float*>(ws + L.off_scores) : nullptr;
  p.weights = key_weights;
  p.score_len = L.score_len;
  p.block_log = __builtin_ctz(static_cast<unsigned>(block));
  p.nblk = static_cast<int>((cache_len + block - 1) / block);
  p.c = scale_log2;
  const int64_t out_rows = static_cast<int64_t>(batch) * heads_q;
  p.weight_wgs = static_cast<int>((cache_len + kWeightKeys - 1) / kWeightKeys);
  const int64_t merge_grid = out_rows + (key_weights != nullptr ? pairs * p.weight_wgs : 0);
  if (merge_grid > ((int64_t{1} << 32) - 1) / 256) return invalid(n + ": grid too large");
  const hipStream_t st = as_stream(stream);
  const bool inline_plan = batch <= kInlineSeqs && rows <= INT32_MAX;
  if (!inline_plan)
    hipLaunchKernelGGL(decode_plan_kernel<CacheDecodeParams>, dim3(1), dim3(kPlanThreads), 0, st, p);
  const int64_t most = pairs * ((cache_len + p.pad + CacheDecodeParams::kMinShare - 1) / CacheDecodeParams::kMinShare);
  const dim3 grid(static_cast<uint32_t>(most < 2 * p.target ? most : 2 * p.target));
  const bool streamed = rows * 2 * kD >= kStreamBytes;
  if (codes == kE4m3)
    launch_split<kE4m3>(inline_plan, streamed, grid, st, p);
  else
    launch_split<kInt8>(inline_plan, streamed, grid, st, p);
  hipLaunchKernelGGL(cache_merge_kernel, dim3(static_cast<uint32_t>(merge_grid)), dim3(256), 0, st, p);
  return launch_status(n.c_str());
}

}  // extern "C"
