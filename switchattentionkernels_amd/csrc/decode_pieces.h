// What a workgroup of a decode over bf16 caches does with its share of the line of
// routed keys (decode_line.h): the kernel body that the decode over whole caches and the
// one behind shared prefixes have in common.
#pragma once

#include "decode_line.h"

namespace swattn {
namespace {

constexpr int kDecWaves = 4;         // waves per workgroup
constexpr int kMaxG = 8;
constexpr uint32_t kPairPad = 192;   // a pair's start, in keys

struct RowParams : DecodeCommon {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  float c;           // sm_scale * log2(e)
};

// One partial (maximum, sum, unnormalised output) per wave and head.
template <int G>
struct PieceLds {
  float m[kDecWaves][G], l[kDecWaves][G];
  float acc[kDecWaves][G][kD];
};

__device__ __forceinline__ float bf(uint32_t bits16) { return __uint_as_float(bits16 << 16); }

// Sum over each row of 16 lanes, every lane getting the row's sum, with DPP
// moves only (no LDS round trip): swap neighbours, swap pairs, then add the
// mirror image within 8 and within 16 lanes.
__device__ __forceinline__ float row16_sum(float x) {
  constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kXor1, 0xf, 0xf, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kXor2, 0xf, 0xf, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kHalfMirror, 0xf, 0xf, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kMirror, 0xf, 0xf, false));
  return x;
}

// One workgroup per share of the line; it takes its pairs one after the other,
// a piece of each.  Lane l works on the keys of key group kg = l / 16 and on
// dims 8*(l%16) .. +7: wave w takes the keys 16*i + 4*w + kg of its piece, so
// the four waves sweep the piece together, four keys per wave per step.
// Each key group keeps its own online-softmax state (running max m, sum l,
// unnormalised sum acc of p * v) for every head of the group; the max moves
// only when a score exceeds it by more than 8 in the exp2 domain, so the
// state is rarely rescaled (the prefill kernel's rule).  The groups and
// waves are combined at the end into one partial per piece, in slot
// blockIdx.x + (pair's rank): both only grow along the line, one of them at
// every step from piece to piece, so that no two pieces share a slot and a
// pair's slots are consecutive.
//
// kStrict (the parameters' kKeepNan): scores of -inf ahead of a lane's first finite one
// weigh nothing, a NaN score shows in the row whatever the others are, and values of
// rows outside the piece (which are read as its nearest row) are not looked at.
template <int G, bool kInline, class P>
__device__ __forceinline__ void decode_pieces(const P& p, uint32_t wg, const SplitStart& st, const SeqEntry* s_ent,
                                              PieceLds<G>& lds) {
  constexpr bool kStrict = P::kKeepNan;
  // Workgroup-uniform walk over the pieces, in scalar registers.
  auto uniform = [](uint32_t x) { return static_cast<int>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); };
  int r = uniform(st.r), kvh = uniform(st.kvh);
  uint32_t key = uniform(st.key);
  uint32_t left = uniform(st.take);   // positions of the line this workgroup still has to take
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int kg = lane >> 4, ds = lane & 15;
  const int64_t row_stride = static_cast<int64_t>(p.hkv) * kD;   // elements per cache row
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
    const int64_t slot = static_cast<int64_t>(wg) + static_cast<int64_t>(r) * p.hkv + kvh;
    // Piece [k0, k1) of the pair's keys.
    const int k0 = uniform(e.lo) + static_cast<int>(key), k1 = k0 + static_cast<int>(min(took, n - key));
    // Q rows of the group: dims 8*ds .. +7 of each head, in fp32, pre-scaled
    // by c so that a dot product is already the exp2-domain score.
    float qv[G][8];
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const uint4 u = *reinterpret_cast<const uint4*>(
          p.q + (static_cast<int64_t>(b) * p.hq + kvh * G + h) * kD + 8 * ds);
      const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qv[h][2 * i] = bf(x[i] & 0xffffu) * p.c;
        qv[h][2 * i + 1] = bf(x[i] >> 16) * p.c;
      }
    }
    const uint16_t* kb = p.k + static_cast<int64_t>(b) * p.cache_len * row_stride + kvh * kD + 8 * ds;
    const uint16_t* vb = p.v + static_cast<int64_t>(b) * p.cache_len * row_stride + kvh * kD + 8 * ds;
    // Keys of this lane: first = k0 aligned down to 16, then every 16.
    const int base = (k0 & ~15) + 4 * wave + kg;
    const int steps = (k1 - (k0 & ~15) + 15) >> 4;
    // Loads run kPf steps ahead of the compute (a ring of registers, the loop
    // unrolled by kPf so that every slot is static): one step alone is four
    // keys per wave, far too little to cover HBM latency.
    constexpr int kPf = G <= 4 ? 8 : 4;
    uint4 kr[kPf], vr[kPf];
    auto load = [&](int i, uint4& kv, uint4& vv) {
      const int kk = min(max(base + 16 * i, k0), k1 - 1);   // in bounds; masked below
      kv = *reinterpret_cast<const uint4*>(kb + kk * row_stride);
      vv = *reinterpret_cast<const uint4*>(vb + kk * row_stride);
    };
#pragma unroll
    for (int j = 0; j < kPf; ++j) load(j, kr[j], vr[j]);
    float m[G], l[G], acc[G][8];
#pragma unroll
    for (int h = 0; h < G; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[h][i] = 0.f;
    }
    for (int i0 = 0; i0 < steps; i0 += kPf) {
#pragma unroll
      for (int j = 0; j < kPf; ++j) {
        const int i = i0 + j;
        if (i >= steps) break;
        const int kk = base + 16 * i;
        const bool live = kk >= k0 && kk < k1;
        const uint32_t kx[4] = {kr[j].x, kr[j].y, kr[j].z, kr[j].w};
        float s[G];
#pragma unroll
        for (int h = 0; h < G; ++h) s[h] = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const float a0 = bf(kx[d] & 0xffffu), a1 = bf(kx[d] >> 16);
#pragma unroll
          for (int h = 0; h < G; ++h)
            s[h] = __builtin_fmaf(a1, qv[h][2 * d + 1], __builtin_fmaf(a0, qv[h][2 * d], s[h]));
        }
        bool moved = false;
#pragma unroll
        for (int h = 0; h < G; ++h) {
          s[h] = row16_sum(s[h]);
          if (!live) s[h] = -INFINITY;
          moved = moved || (s[h] - m[h] > 8.0f);
        }
        if (__builtin_amdgcn_ballot_w64(moved)) {   // rare: move the maxima, rescale
#pragma unroll
          for (int h = 0; h < G; ++h) {
            const float mn = s[h] - m[h] > 8.0f ? s[h] : m[h];
            const float a = mn == m[h] ? 1.0f : __builtin_amdgcn_exp2f(m[h] - mn);
            m[h] = mn;
            l[h] *= a;
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[h][d] *= a;
          }
        }
        uint32_t vx[4] = {vr[j].x, vr[j].y, vr[j].z, vr[j].w};
        if constexpr (kStrict) {
#pragma unroll
          for (int d = 0; d < 4; ++d) vx[d] = live ? vx[d] : 0u;
        }
#pragma unroll
        for (int h = 0; h < G; ++h) {
          const float from = kStrict && m[h] == -INFINITY ? 0.f : m[h];
          const float pr = live ? __builtin_amdgcn_exp2f(s[h] - from) : 0.f;
          l[h] += pr;
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            acc[h][2 * d] = __builtin_fmaf(pr, bf(vx[d] & 0xffffu), acc[h][2 * d]);
            acc[h][2 * d + 1] = __builtin_fmaf(pr, bf(vx[d] >> 16), acc[h][2 * d + 1]);
          }
        }
        load(i + kPf, kr[j], vr[j]);   // refill the slot; past the end: clamped, never used
      }
    }
    // Combine the four key groups of the wave (lanes l, l^16, l^32, l^48 hold
    // the same dims of different keys).
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float mm = m[h];
      mm = fmaxf(mm, __shfl_xor(mm, 16));
      mm = fmaxf(mm, __shfl_xor(mm, 32));
      // (kStrict: where no score is finite, the sums are 0 or NaN, and stay.)
      const float a = mm == -INFINITY ? (kStrict ? 1.f : 0.f) : exp2f(m[h] - mm);
      float lh = l[h] * a;
      lh += __shfl_xor(lh, 16);
      lh += __shfl_xor(lh, 32);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        float x = acc[h][d] * a;
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        if (kg == 0) lds.acc[wave][h][8 * ds + d] = x;
      }
      if (lane == 0) {
        lds.m[wave][h] = mm;
        lds.l[wave][h] = lh;
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
      for (int w = 0; w < kDecWaves; ++w) mm = fmaxf(mm, lds.m[w][h]);
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) {
        if constexpr (kStrict)
          a += (mm == -INFINITY ? 1.f : exp2f(lds.m[w][h] - mm)) * lds.acc[w][h][d];
        else if (lds.m[w][h] != -INFINITY)
          a += exp2f(lds.m[w][h] - mm) * lds.acc[w][h][d];
      }
      po[i] = a;
    }
    if (tid < G) {
      float mm = -INFINITY, lh = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) mm = fmaxf(mm, lds.m[w][tid]);
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) {
        if constexpr (kStrict)
          lh += (mm == -INFINITY ? 1.f : exp2f(lds.m[w][tid] - mm)) * lds.l[w][tid];
        else if (lds.m[w][tid] != -INFINITY)
          lh += exp2f(lds.m[w][tid] - mm) * lds.l[w][tid];
      }
      pml[2 * tid] = mm;
      pml[2 * tid + 1] = lh;
    }
    }
    // The rest of the share continues at the start of the next pair (the
    // share ends inside this one otherwise).
    if (left == 0u) return;
    key = 0;
    if (++kvh == p.hkv) {
      kvh = 0;
      ++r;
    }
    __syncthreads();   // the next piece's combine writes the same LDS
  }
}

}  // namespace
}  // namespace swattn
