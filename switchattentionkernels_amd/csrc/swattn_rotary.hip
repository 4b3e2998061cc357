// Per-head norms and position rotation of queries and keys in one pass, forward and
// backward, for gfx950 (include/swattn_rotary.h).  No counterpart in the reference.
//
//   r = 1 / sqrt(mean(x^2) + eps),  u = r x,  y = w u   (no weight: y = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = inv_freq[i] * position
//   backward, g = dy rotated by -t:  dw = sum g u,  dx = r (g w - u mean(g w u))
//
// HBM-bound: 512 bytes per head row forward, 768 backward (512 without a norm) against
// about a dozen operations per value.  A wave takes eight head rows of a token at once (a
// pass), eight lanes per row; a lane holds two 16-byte chunks of its row whose dims form
// whole pairs, so that the rotation needs no exchange between lanes and the norm a sum over
// eight lanes.  The token's angles are the same for all its heads: each lane computes one
// frequency's sine and cosine, and the lanes pick up the eight that their dims need from
// LDS, as the norms' weights: kept in registers, both cost a third of the waves.
// The grid is what the chip takes at once.  Waves go over whole tokens in rounds, side by
// side, and share out the passes of the tokens that are left: with tokens alone a batch of
// 5998 left a third of the waves idle, with one run of passes per wave B1 S16384 Hq32/Hkv8
// took 72 us instead of 69.  Rows are read one pass ahead.
//
// Measured, as a large copy's 5.2 TB/s goes (a copy of 74 MB: 5.0): rotations of strided
// rows B1 S16384 Hq32/Hkv8 62.7 us (5.4 TB/s), B2 S2999 Hq40/Hkv8 30.0 (4.9); backward of
// S16384 with norms 92 us (5.4 TB/s), of B2 S4096 without 28.9; appends of B8 T517 Hq64/Hkv8
// 33.5 (4.7), of 64 single tokens 6.6, bound by dependent latencies and the host's call.
// One pass at a time without reading ahead, angles and weights in registers: 71, 42, 117, 42,
// 50 and 7.5.
//
// Angles are exact where fp32 products are not (a position of 2^17 times a frequency of
// 1 is off by up to 2^-8 in fp32): a frequency is held as a 64-bit fixed-point fraction
// of turns per position, and the product with the position is taken mod 2^64, which drops
// whole turns: an angle is off by 2^-65 turns per position.

#include <math.h>

#include <string>

#include "common.h"
#include "swattn_rotary.h"

namespace swattn {
namespace {

constexpr int kD = 128;
constexpr int kWaves = 4;          // waves per workgroup
constexpr int kRowsAtOnce = 8;     // head rows that a wave takes at once
constexpr int kGroupsPerCu = 5;    // workgroups that a CU takes at once (4 and 6: within 2 %)
constexpr int kBackPerCu = 3;      // and of the backward (4: S16384 108 us instead of 101, 5 spill: 187)
// Calls that move more than kStreamBytes go past the 256 MB memory-side cache, the forward in
// both directions (S16384 Hq32/Hkv8 69.5 -> 62.5 us, B2 S2999 Hq40/Hkv8 33.4 -> 29.9; B1 S2729
// Hq32/Hkv8, 56 MB that a projection may have left there, 11.0, streamed 13.5), the backward with
// what it writes (B1 S3077 Hq40/Hkv8 30.6 -> 27.1), and with what it reads if that alone fills the
// cache (S16384 98 -> 93.5; S3077 27.1 -> 32).
constexpr int64_t kStreamBytes = 96 << 20, kCacheBytes = 256 << 20;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Rows {
  const uint16_t* p;
  int64_t sb, ss, sh;   // strides of batch, token and head, in elements
};

struct Angles {
  const int32_t* positions;   // [axes][batch * seq]
  const void* freq;
  int f64, count, axes;
  int ends[SWATTN_ROTARY_MAX_AXES - 1];   // frequencies before each axis but the first
};

// How the waves share the tokens' passes over eight head rows: whole tokens in rounds,
// neighbours to neighbours, then the passes of the tokens that are left in equal shares.
struct Shares {
  int waves, rounds;
  int64_t each;   // passes of what is left, and one more for the first `more` waves
  int more;
};
struct Part {     // passes [pass, end) of a token; end 0: none
  int token, pass, end;
};
struct Walk {
  uint32_t token;   // of the next round
  int rounds, left_token, left_pass;
  int64_t left;
};
__device__ __forceinline__ Walk walk_of(const Shares& s, int wave, int passes) {
  const int64_t from = wave * s.each + min(wave, s.more);   // below waves * passes
  const int token = from >> 32 == 0 ? static_cast<int>(static_cast<uint32_t>(from) / static_cast<uint32_t>(passes))
                                    : static_cast<int>(from / passes);
  return Walk{static_cast<uint32_t>(wave), s.rounds, s.waves * s.rounds + token,
              static_cast<int>(from - static_cast<int64_t>(token) * passes), s.each + (wave < s.more ? 1 : 0)};
}
__device__ __forceinline__ Part advance(Walk& w, const Shares& s, int passes) {
  if (w.rounds > 0) {
    const int token = static_cast<int>(w.token);
    --w.rounds;
    w.token += s.waves;
    return Part{token, 0, passes};
  }
  if (w.left == 0) return Part{0, 0, 0};
  const Part x{w.left_token, w.left_pass, static_cast<int>(min(static_cast<int64_t>(passes), w.left_pass + w.left))};
  w.left -= x.end - x.pass;
  ++w.left_token;
  w.left_pass = 0;
  return x;
}

struct RotaryParams {
  Rows q, k, v;
  Angles angles;
  const void* q_weight;
  const void* k_weight;
  int weight_bf16;
  float eps;
  uint16_t* q_out;
  uint16_t* k_out;    // rows, or the cache
  uint16_t* v_out;    // the cache
  const int32_t* lens;
  const int32_t* counts;
  int32_t* lens_out;
  int64_t cache_len;
  int batch, seq, tokens, hq, hkv;
  Shares shares;
};

// Turns per position as a 64-bit fraction: f / (2 pi), with 1 / (2 pi) and the product
// in two doubles each, its whole turns dropped.
__device__ __forceinline__ uint64_t fixed_turns(double f) {
  constexpr double kInv2Pi = 0x1.45f306dc9c883p-3, kInv2PiLow = -0x1.6b01ec5417056p-57;
  const double y = f * kInv2Pi;
  const double low = __builtin_fma(f, kInv2PiLow, __builtin_fma(f, kInv2Pi, -y));
  const double t = (y - __builtin_rint(y)) * 0x1p32;   // exact
  const double whole = __builtin_rint(t);
  const int64_t rest = static_cast<int64_t>(__builtin_rint(((t - whole) + low * 0x1p32) * 0x1p32));
  return (static_cast<uint64_t>(static_cast<int64_t>(whole)) << 32) + static_cast<uint64_t>(rest);
}

// Sine and cosine of an angle in 2^-64 turns: the nearest quarter turn, and the Taylor
// series of what is left, at most pi / 4 (the next terms are below 2^-29).  What is left
// enters with fp32's bits however small it is: its upper 32 bits, rounded, and what that
// leaves.  (The upper 32 bits alone, steps of 1.5e-9 radians, were 1 % of the sine of a
// frequency of 1e-8 at position 1.)
__device__ __forceinline__ void sine_cosine(uint64_t turns, float& s, float& c) {
  const uint32_t quarter = static_cast<uint32_t>((turns + 0x2000000000000000u) >> 62);
  const uint64_t rest = turns - (static_cast<uint64_t>(quarter) << 62);
  const int32_t high = static_cast<int32_t>((rest + 0x80000000u) >> 32), low = static_cast<int32_t>(rest);
  constexpr float kStep = 1.46291807926716e-9f;   // 2 pi / 2^32
  const float x = __builtin_fmaf(static_cast<float>(low), kStep * 0x1p-32f, static_cast<float>(high) * kStep);
  const float z = x * x;
  float a = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);   // 1 / 9!, 1 / 7!, ..
  a = __builtin_fmaf(z, a, 8.33333333e-3f);
  a = __builtin_fmaf(z, a, -1.66666667e-1f);
  a = __builtin_fmaf(x * z, a, x);
  float b = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);   // 1 / 10!, 1 / 8!, ..
  b = __builtin_fmaf(z, b, -1.38888889e-3f);
  b = __builtin_fmaf(z, b, 4.16666667e-2f);
  b = __builtin_fmaf(z, b, -0.5f);
  b = __builtin_fmaf(z, b, 1.0f);
  s = quarter & 1u ? b : a;
  c = quarter & 1u ? a : b;
  if (quarter & 2u) s = -s;
  if ((quarter + 1u) & 2u) c = -c;
}

// What a lane knows for all tokens: the fraction of its frequency (frequency `lane`),
// its axis, and where its two chunks lie in a row.
struct Lane {
  uint64_t turns;
  int axis;
  bool nan;
  bool turned;   // its dims are among those that are rotated
  int a, b;      // first dims of its chunks: pairs lie across them, or inside each
};
template <bool kPairs>
__device__ __forceinline__ Lane lane_setup(const Angles& g, int lane) {
  Lane o;
  const int i = min(lane, g.count - 1), l = lane & 7;
  o.axis = 0;
#pragma unroll
  for (int x = 0; x < SWATTN_ROTARY_MAX_AXES - 1; ++x) o.axis += x + 1 < g.axes && i >= g.ends[x] ? 1 : 0;
  o.turned = 8 * l < g.count;
  const bool beside = kPairs || !o.turned;   // dims behind the rotated ones: what is left, in order
  o.a = beside ? 16 * l : 8 * l;
  o.b = beside ? o.a + 8 : o.a + g.count;
  return o;
}
__device__ __forceinline__ void lane_turns(const Angles& g, int lane, Lane& o) {
  const int i = min(lane, g.count - 1);
  const double f = g.f64 ? static_cast<const double*>(g.freq)[i] : static_cast<double>(static_cast<const float*>(g.freq)[i]);
  o.nan = !(__builtin_fabs(f) < 0x1p40);
  o.turns = fixed_turns(o.nan ? 0.0 : f);
}

__device__ __forceinline__ int token_position(const Angles& g, const Lane& o, int64_t token, int tokens) {
  return g.positions[static_cast<int64_t>(o.axis) * tokens + token];
}

// Cosines and sines of a token's frequencies, in the wave's own LDS words (a wave's LDS
// operations complete in order).
__device__ __forceinline__ void token_turn(const Lane& o, int pos, int lane, float (*lds)[64]) {
  const uint64_t at = o.turns * static_cast<uint64_t>(static_cast<int64_t>(pos));
  float s, c;
  sine_cosine(at, s, c);
  __builtin_amdgcn_wave_barrier();
  lds[0][lane] = o.nan ? NAN : c;
  lds[1][lane] = o.nan ? NAN : s;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// x: dims a .. a + 7, then b .. b + 7, rotated by +t or -t.
template <bool kPairs, bool kBack>
__device__ __forceinline__ void rotate(const Lane& o, const float (*lds)[64], int lane, float (&x)[16]) {
  if (!o.turned) return;
  const int first = 8 * (lane & 7);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = kPairs ? 2 * e : e, j = kPairs ? 2 * e + 1 : e + 8;
    const float c = lds[0][first + e], s = kBack ? -lds[1][first + e] : lds[1][first + e];
    const float a = x[i], b = x[j];
    x[i] = a * c - b * s;
    x[j] = b * c + a * s;
  }
}

// Sum over the eight lanes of a row, the same in each.
__device__ __forceinline__ float row_sum(float x) {
  constexpr int kHalfMirror = 0x141;
  x += lane_move<kXor1>(x);
  x += lane_move<kXor2>(x);
  return x + lane_move<kHalfMirror>(x);
}

struct Chunks {
  u32x4 a, b;
};
template <bool kStream>
__device__ __forceinline__ void load_chunks(const uint16_t* row, const Lane& o, Chunks& c) {
  const u32x4 *a = reinterpret_cast<const u32x4*>(row + o.a), *b = reinterpret_cast<const u32x4*>(row + o.b);
  c.a = kStream ? __builtin_nontemporal_load(a) : *a;
  c.b = kStream ? __builtin_nontemporal_load(b) : *b;
}
template <bool kStream>
__device__ __forceinline__ void store_chunks(uint16_t* row, const Lane& o, const Chunks& c) {
  u32x4 *a = reinterpret_cast<u32x4*>(row + o.a), *b = reinterpret_cast<u32x4*>(row + o.b);
  if constexpr (kStream) {
    __builtin_nontemporal_store(c.a, a);
    __builtin_nontemporal_store(c.b, b);
  } else {
    *a = c.a;
    *b = c.b;
  }
}
__device__ __forceinline__ void unpack(const Chunks& c, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(c.a[i] << 16);
    x[2 * i + 1] = __uint_as_float(c.a[i] & 0xffff0000u);
    x[8 + 2 * i] = __uint_as_float(c.b[i] << 16);
    x[8 + 2 * i + 1] = __uint_as_float(c.b[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
template <bool kStream>
__device__ __forceinline__ void store_row(uint16_t* row, const Lane& o, const float (&x)[16]) {
  store_chunks<kStream>(row, o,
                        Chunks{u32x4{pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7])},
                               u32x4{pack(x[8], x[9]), pack(x[10], x[11]), pack(x[12], x[13]), pack(x[14], x[15])}});
}

// A tensor's weights in LDS, by the workgroup's first or second 128 threads.
__device__ __forceinline__ void stage_weights(const void* w, int bf16, int d, float* lds) {
  if (w == nullptr) return;
  lds[d] = bf16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(w)[d]) << 16) : static_cast<const float*>(w)[d];
}
__device__ __forceinline__ void load_weights(const float* lds, const Lane& o, float (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = lds[o.a + i];
    w[8 + i] = lds[o.b + i];
  }
}

// x becomes x / sqrt(mean(x^2) + eps); returns what it was multiplied by.  The root is the
// hardware's, within one last place, which takes no denormal number.  A row whose mean
// square leaves [2^-96, 2^120) (finite rows of bf16 may have 2^-266 to 2^256) is scaled by a power of
// two first, so that its squares and their sum stay fp32 numbers.
__device__ __forceinline__ float normalise(float (&x)[16], float eps) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = __builtin_fmaf(x[i], x[i], s);
  const float m = __builtin_fmaf(row_sum(s), 1.0f / kD, eps);
  float r = __builtin_amdgcn_rsqf(m), by = 1.0f;
  if (!(m >= 0x1p-96f && m < 0x1p120f)) {   // the same in a row's lanes; rare
    by = m < 1.0f ? 0x1p100f : 0x1p-68f;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] *= by;
      s = __builtin_fmaf(x[i], x[i], s);
    }
    r = __builtin_amdgcn_rsqf(__builtin_fmaf(row_sum(s), 1.0f / kD, eps * by * by));
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] *= r;
  return r * by;
}

// A wave goes through its share of the passes: a token's q rows, then its k rows, then its
// v rows, which are copied.  A pass's rows are read one pass ahead, a token's positions one
// token ahead.
template <bool kPairs, bool kAppend, bool kStream>
__global__ __launch_bounds__(64 * kWaves, kGroupsPerCu) void rotary_kernel(const RotaryParams p) {
  __shared__ float s_turn[kWaves][2][64];
  __shared__ float s_weight[2][kD];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if constexpr (kAppend) {
    for (int b = blockIdx.x * blockDim.x + tid; b < p.batch; b += gridDim.x * blockDim.x) {
      const int64_t len = min(max(static_cast<int64_t>(p.lens[b]), int64_t{0}), p.cache_len);
      const int count = p.counts == nullptr ? p.seq : min(max(p.counts[b], 0), p.seq);
      p.lens_out[b] = static_cast<int32_t>(min(len + count, p.cache_len));
    }
  }
  const int q_passes = (p.hq + kRowsAtOnce - 1) / kRowsAtOnce, k_passes = (p.hkv + kRowsAtOnce - 1) / kRowsAtOnce;
  const int passes = q_passes + (kAppend ? 2 : 1) * k_passes;
  Walk walk = walk_of(p.shares, blockIdx.x * kWaves + wave, passes);
  Lane o = lane_setup<kPairs>(p.angles, lane);
  auto tensor = [&](int pass) { return pass < q_passes ? 0 : pass < q_passes + k_passes ? 1 : 2; };
  auto head = [&](int pass, int x) {
    return (pass - (x == 0 ? 0 : x == 1 ? q_passes : q_passes + k_passes)) * kRowsAtOnce + (lane >> 3);
  };
  auto load = [&](int b, int s, int pass, Chunks& c) {
    const int x = tensor(pass), h = head(pass, x);
    const Rows& in = x == 0 ? p.q : x == 1 ? p.k : p.v;
    if (h < (x == 0 ? p.hq : p.hkv)) load_chunks<kStream>(in.p + b * in.sb + s * in.ss + h * in.sh, o, c);
  };
  Part now = advance(walk, p.shares, passes);
  int b = 0, s = 0, pos = 0;
  Chunks next;
  if (now.end > 0) {
    b = now.token / p.seq;
    s = now.token - b * p.seq;
    load(b, s, now.pass, next);
    pos = token_position(p.angles, o, now.token, p.tokens);
  }
  stage_weights(tid < kD ? p.q_weight : p.k_weight, p.weight_bf16, tid & (kD - 1), s_weight[tid / kD]);
  lane_turns(p.angles, lane, o);
  __syncthreads();
  while (now.end > 0) {
    token_turn(o, pos, lane, s_turn[wave]);
    int64_t at = now.token;       // of the row that K (and V) go to, in k_out
    bool live = true;
    if constexpr (kAppend) {
      const int64_t len = min(max(static_cast<int64_t>(p.lens[b]), int64_t{0}), p.cache_len);
      live = len + s < p.cache_len && (p.counts == nullptr || s < p.counts[b]);
      at = b * p.cache_len + len + s;
    }
    const Part then = advance(walk, p.shares, passes);
    const int b1 = b, s1 = s;
    if (then.end > 0) {
      b = then.token / p.seq;
      s = then.token - b * p.seq;
      pos = token_position(p.angles, o, then.token, p.tokens);
    }
    for (int pass = now.pass; pass < now.end; ++pass) {
      const Chunks c = next;
      if (pass + 1 < now.end) {
        if (live || pass + 1 < q_passes) load(b1, s1, pass + 1, next);
      } else if (then.end > 0) {
        load(b, s, then.pass, next);
      }
      const int which = tensor(pass), h = head(pass, which);
      if (h >= (which == 0 ? p.hq : p.hkv) || !(which == 0 || live)) continue;
      uint16_t* row = which == 0 ? p.q_out + (static_cast<int64_t>(now.token) * p.hq + h) * kD
                                 : (which == 1 ? p.k_out : p.v_out) + (at * p.hkv + h) * kD;
      if (which == 2) {
        store_chunks<kStream>(row, o, c);
        continue;
      }
      float x[16];
      unpack(c, x);
      if ((which == 0 ? p.q_weight : p.k_weight) != nullptr) {
        float w[16];
        load_weights(s_weight[which], o, w);
        normalise(x, p.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= w[i];
      }
      rotate<kPairs, false>(o, s_turn[wave], lane, x);
      store_row<kStream>(row, o, x);
    }
    now = then;
  }
}

struct BackwardParams {
  Rows x[2];                    // q, k
  Angles angles;
  const uint16_t* grad[2];      // contiguous
  const void* weight[2];
  uint16_t* dx[2];
  float* part[2];               // [workgroups][128] sums of g u, or null
  int heads[2], groups[2];      // workgroups of each tensor
  Shares shares[2];
  int weight_bf16;
  float eps;
  int seq, tokens;
};

// The first groups[0] workgroups take q's rows, the others k's; a wave's loop is the
// forward's.
template <bool kPairs, bool kStreamIn, bool kStreamOut>
__global__ __launch_bounds__(64 * kWaves, kBackPerCu) void rotary_backward_kernel(const BackwardParams p) {
  __shared__ float s_turn[kWaves][2][64];
  __shared__ float s_weight[kD];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int which = static_cast<int>(blockIdx.x) < p.groups[0] ? 0 : 1;
  const int group = blockIdx.x - (which ? p.groups[0] : 0);
  const Rows in = p.x[which];
  const uint16_t* grad = p.grad[which];
  const void* weight = p.weight[which];
  float* part = p.part[which];
  const int heads = p.heads[which], passes = (heads + kRowsAtOnce - 1) / kRowsAtOnce;
  Lane o = lane_setup<kPairs>(p.angles, lane);
  struct Both {
    Chunks g, x;
  };
  auto load = [&](int token, int b, int s, int pass, Both& c) {
    const int h = pass * kRowsAtOnce + (lane >> 3);
    if (h >= heads) return;
    load_chunks<kStreamIn>(grad + (static_cast<int64_t>(token) * heads + h) * kD, o, c.g);
    if (weight != nullptr) load_chunks<kStreamIn>(in.p + b * in.sb + s * in.ss + h * in.sh, o, c.x);
  };
  float dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f;
  const Shares& shares = p.shares[which];
  Walk walk = walk_of(shares, group * kWaves + wave, passes);
  Part now = advance(walk, shares, passes);
  int b = 0, s = 0, pos = 0;
  Both next;
  if (now.end > 0) {
    b = now.token / p.seq;
    s = now.token - b * p.seq;
    load(now.token, b, s, now.pass, next);
    pos = token_position(p.angles, o, now.token, p.tokens);
  }
  if (tid < kD) stage_weights(weight, p.weight_bf16, tid, s_weight);
  lane_turns(p.angles, lane, o);
  __syncthreads();
  while (now.end > 0) {
    token_turn(o, pos, lane, s_turn[wave]);
    const Part then = advance(walk, shares, passes);
    const int b1 = b, s1 = s;
    if (then.end > 0) {
      b = then.token / p.seq;
      s = then.token - b * p.seq;
      pos = token_position(p.angles, o, then.token, p.tokens);
    }
    for (int pass = now.pass; pass < now.end; ++pass) {
      const Both c = next;
      if (pass + 1 < now.end)
        load(now.token, b1, s1, pass + 1, next);
      else if (then.end > 0)
        load(then.token, b, s, then.pass, next);
      const int h = pass * kRowsAtOnce + (lane >> 3);
      if (h >= heads) continue;
      float g[16];
      unpack(c.g, g);
      rotate<kPairs, true>(o, s_turn[wave], lane, g);
      if (weight != nullptr) {
        float u[16], w[16];
        unpack(c.x, u);
        load_weights(s_weight, o, w);
        const float r = normalise(u, p.eps);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          dw[i] = __builtin_fmaf(g[i], u[i], dw[i]);
          g[i] *= w[i];
          dot = __builtin_fmaf(g[i], u[i], dot);
        }
        dot = row_sum(dot) * (1.0f / kD);
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = r * __builtin_fmaf(-u[i], dot, g[i]);
      }
      store_row<kStreamOut>(p.dx[which] + (static_cast<int64_t>(now.token) * heads + h) * kD, o, g);
    }
    now = then;
  }
  if (part == nullptr) return;   // uniform
  // Sums over the wave's eight rows, then over the waves.
  __shared__ float s_dw[kWaves][kD];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x = with_lane32(with_lane16(dw[i] + lane_move<kTurn8>(dw[i]), Add()), Add());
    if (lane < 8) s_dw[wave][i < 8 ? o.a + i : o.b + i - 8] = x;
  }
  __syncthreads();
  if (tid < kD) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) x += s_dw[i][tid];
    part[static_cast<int64_t>(group) * kD + tid] = x;
  }
}

// Sums over the workgroups' partials, 8 dims per workgroup: thread (g, d) takes every
// 32nd partial from g on, then the 32 sums are added in order.
constexpr int kSumDims = 8;
struct SumParams {
  const float* part[2];
  void* out[2];
  int groups[2];
  int bf16;
};
__global__ __launch_bounds__(256) void rotary_sum_kernel(const SumParams p) {
  __shared__ float s_sum[32][kSumDims];
  const int which = blockIdx.y;
  if (p.out[which] == nullptr) return;   // uniform
  const int d = threadIdx.x & (kSumDims - 1), g = threadIdx.x / kSumDims;
  const int dim = blockIdx.x * kSumDims + d;
  float x = 0.f;
#pragma unroll 8
  for (int i = g; i < p.groups[which]; i += 32) x += p.part[which][static_cast<int64_t>(i) * kD + dim];
  s_sum[g][d] = x;
  __syncthreads();
  if (g != 0) return;
  x = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) x += s_sum[i][d];
  if (p.bf16)
    static_cast<uint16_t*>(p.out[which])[dim] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  else
    static_cast<float*>(p.out[which])[dim] = x;
}

int cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    return 256;
  return n;
}


int64_t passes_of(int64_t heads) { return (heads + kRowsAtOnce - 1) / kRowsAtOnce; }

Shares shares_of(int64_t tokens, int64_t passes, int64_t groups) {
  const int64_t waves = groups * kWaves, rounds = tokens / waves, left = (tokens - rounds * waves) * passes;
  return Shares{static_cast<int>(waves), static_cast<int>(rounds), left / waves, static_cast<int>(left % waves)};
}

// Workgroups of the backward for q and for k: as their rows, at least one each.
void backward_groups(int64_t tokens, int64_t hq, int64_t hkv, int (&groups)[2]) {
  const int64_t pq = passes_of(hq), pk = passes_of(hkv), most = int64_t{kBackPerCu} * cus();
  const int64_t q = most * pq / (pq + pk), k = most - q;
  auto within = [&](int64_t x, int64_t passes) {
    const int64_t need = (tokens * passes + kWaves - 1) / kWaves;
    return static_cast<int>(x < 1 || need < 1 ? 1 : x > need ? need : x);
  };
  groups[0] = within(q, pq);
  groups[1] = within(k, pk);
}

bool rows_ok(const void* p, const int64_t* strides, Rows& out) {
  if (p == nullptr || strides == nullptr || !aligned16(p)) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0) return false;
  out = Rows{static_cast<const uint16_t*>(p), strides[0], strides[1], strides[2]};
  return true;
}

int check_shape(const std::string& n, int32_t batch, int64_t seq, int32_t heads_q, int32_t heads_kv, int32_t head_dim) {
  if (head_dim != kD) return invalid(n + ": head_dim must be 128");
  if (batch < 1 || seq < 0 || heads_q < 1 || heads_kv < 1) return invalid(n + ": bad shape");
  if (heads_q > 65535 || heads_kv > 65535 || seq > INT32_MAX || batch * seq > INT32_MAX)
    return invalid(n + ": batch * seq or heads too large");
  return SWATTN_OK;
}

int check_angles(const std::string& n, const int32_t* positions, const void* inv_freq, int32_t freq_f64,
                 const int32_t* sections, int32_t axes, Angles& out) {
  if (positions == nullptr || inv_freq == nullptr || sections == nullptr) return invalid(n + ": null pointer");
  if (axes < 1 || axes > SWATTN_ROTARY_MAX_AXES) return invalid(n + ": axes must be 1 to 4");
  int64_t count = 0;
  out = Angles{positions, inv_freq, freq_f64 != 0, 0, axes, {0, 0, 0}};
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 1) return invalid(n + ": sections must be positive");
    count += sections[i];
    if (i < SWATTN_ROTARY_MAX_AXES - 1) out.ends[i] = static_cast<int>(count);
  }
  if (count % 8 != 0 || count > kD / 2) return invalid(n + ": the number of frequencies must be a multiple of 8 up to 64");
  out.count = static_cast<int>(count);
  return SWATTN_OK;
}

// A pass per wave, or equal shares of the waves that the chip takes at once.
template <bool kAppend>
int launch_rotary(const char* name, bool pairs, RotaryParams& p, void* stream) {
  if (p.tokens == 0 && !kAppend) return SWATTN_OK;
  const int64_t passes = passes_of(p.hq) + (kAppend ? 2 : 1) * passes_of(p.hkv);
  const int64_t most = int64_t{kGroupsPerCu} * cus(), need = (p.tokens * passes + kWaves - 1) / kWaves;
  const int64_t groups = need < 1 ? 1 : need < most ? need : most;
  p.shares = shares_of(p.tokens, passes, groups);
  const dim3 grid(static_cast<uint32_t>(groups));
  const bool stream_past = p.tokens * (p.hq + (kAppend ? 2 : 1) * int64_t{p.hkv}) * (4 * kD) >= kStreamBytes;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, as_stream(stream), p); };
  if (pairs && stream_past)
    launch(rotary_kernel<true, kAppend, true>);
  else if (pairs)
    launch(rotary_kernel<true, kAppend, false>);
  else if (stream_past)
    launch(rotary_kernel<false, kAppend, true>);
  else
    launch(rotary_kernel<false, kAppend, false>);
  return launch_status(name);
}

}  // namespace
}  // namespace swattn

using namespace swattn;

extern "C" {

int swattn_rotary_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                      const int32_t* positions, const void* inv_freq, int32_t freq_f64,
                      const int32_t* sections, int32_t axes, int32_t interleaved, const void* q_weight,
                      const void* k_weight, int32_t weight_bf16, float eps, void* q_out, void* k_out,
                      int32_t batch, int64_t seq, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                      void* stream) {
  const char* name = "swattn_rotary_fwd";
  const std::string n(name);
  int st = check_shape(n, batch, seq, heads_q, heads_kv, head_dim);
  RotaryParams p{};
  if (st == SWATTN_OK) st = check_angles(n, positions, inv_freq, freq_f64, sections, axes, p.angles);
  if (st != SWATTN_OK) return st;
  if (!rows_ok(q, q_strides, p.q) || !rows_ok(k, k_strides, p.k))
    return invalid(n + ": q and k must be 16-byte aligned, their strides multiples of 8 and not negative");
  if (q_out == nullptr || k_out == nullptr || !aligned16(q_out) || !aligned16(k_out))
    return invalid(n + ": q_out and k_out must be 16-byte aligned");
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.weight_bf16 = weight_bf16;
  p.eps = eps;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.k_out = static_cast<uint16_t*>(k_out);
  p.batch = batch;
  p.seq = static_cast<int>(seq);
  p.tokens = static_cast<int>(batch * seq);
  p.hq = heads_q;
  p.hkv = heads_kv;
  return launch_rotary<false>(name, interleaved != 0, p, stream);
}

int swattn_rotary_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                         const void* v, const int64_t* v_strides, const int32_t* positions,
                         const void* inv_freq, int32_t freq_f64, const int32_t* sections, int32_t axes,
                         int32_t interleaved, const void* q_weight, const void* k_weight,
                         int32_t weight_bf16, float eps, void* q_out, void* k_cache, void* v_cache,
                         const int32_t* cache_lens, const int32_t* counts, int32_t* lens_out,
                         int32_t batch, int64_t seq, int64_t cache_len, int32_t heads_q,
                         int32_t heads_kv, int32_t head_dim, void* stream) {
  const char* name = "swattn_rotary_append";
  const std::string n(name);
  int st = check_shape(n, batch, seq, heads_q, heads_kv, head_dim);
  RotaryParams p{};
  if (st == SWATTN_OK) st = check_angles(n, positions, inv_freq, freq_f64, sections, axes, p.angles);
  if (st != SWATTN_OK) return st;
  if (cache_len < 1 || cache_len > INT32_MAX) return invalid(n + ": bad cache_len");
  if (!rows_ok(q, q_strides, p.q) || !rows_ok(k, k_strides, p.k) || !rows_ok(v, v_strides, p.v))
    return invalid(n + ": q, k and v must be 16-byte aligned, their strides multiples of 8 and not negative");
  if (q_out == nullptr || k_cache == nullptr || v_cache == nullptr || cache_lens == nullptr || lens_out == nullptr)
    return invalid(n + ": null pointer");
  if (!aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache))
    return invalid(n + ": q_out and the caches must be 16-byte aligned");
  if (cache_lens == lens_out) return invalid(n + ": lens_out may not alias cache_lens");
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.weight_bf16 = weight_bf16;
  p.eps = eps;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.k_out = static_cast<uint16_t*>(k_cache);
  p.v_out = static_cast<uint16_t*>(v_cache);
  p.lens = cache_lens;
  p.counts = counts;
  p.lens_out = lens_out;
  p.cache_len = cache_len;
  p.batch = batch;
  p.seq = static_cast<int>(seq);
  p.tokens = static_cast<int>(batch * seq);
  p.hq = heads_q;
  p.hkv = heads_kv;
  return launch_rotary<true>(name, interleaved != 0, p, stream);
}

size_t swattn_rotary_bwd_workspace_bytes(int32_t batch, int64_t seq, int32_t heads_q, int32_t heads_kv) {
  if (check_shape("swattn_rotary_bwd_workspace_bytes", batch, seq, heads_q, heads_kv, kD) != SWATTN_OK) return 0;
  int groups[2];
  backward_groups(batch * seq, heads_q, heads_kv, groups);
  return static_cast<size_t>(groups[0] + groups[1]) * kD * sizeof(float);
}

int swattn_rotary_bwd(const void* grad_q, const void* grad_k, const void* q, const int64_t* q_strides,
                      const void* k, const int64_t* k_strides, const int32_t* positions,
                      const void* inv_freq, int32_t freq_f64, const int32_t* sections, int32_t axes,
                      int32_t interleaved, const void* q_weight, const void* k_weight,
                      int32_t weight_bf16, float eps, void* dq, void* dk, void* dq_weight,
                      void* dk_weight, int32_t batch, int64_t seq, int32_t heads_q, int32_t heads_kv,
                      int32_t head_dim, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "swattn_rotary_bwd";
  const std::string n(name);
  int st = check_shape(n, batch, seq, heads_q, heads_kv, head_dim);
  BackwardParams p{};
  if (st == SWATTN_OK) st = check_angles(n, positions, inv_freq, freq_f64, sections, axes, p.angles);
  if (st != SWATTN_OK) return st;
  if ((q_weight != nullptr && !rows_ok(q, q_strides, p.x[0])) || (k_weight != nullptr && !rows_ok(k, k_strides, p.x[1])))
    return invalid(n + ": q and k must be 16-byte aligned, their strides multiples of 8 and not negative");
  if (grad_q == nullptr || grad_k == nullptr || dq == nullptr || dk == nullptr || !aligned16(grad_q) ||
      !aligned16(grad_k) || !aligned16(dq) || !aligned16(dk))
    return invalid(n + ": the gradients must be 16-byte aligned");
  if ((dq_weight != nullptr && q_weight == nullptr) || (dk_weight != nullptr && k_weight == nullptr))
    return invalid(n + ": a weight's gradient needs the weight");
  const bool sums = dq_weight != nullptr || dk_weight != nullptr;
  if (sums) {
    if (workspace == nullptr || workspace_bytes < swattn_rotary_bwd_workspace_bytes(batch, seq, heads_q, heads_kv)) {
      set_error(n + ": workspace smaller than swattn_rotary_bwd_workspace_bytes()");
      return SWATTN_EWORKSPACE;
    }
    if (!aligned256(workspace)) return invalid(n + ": workspace must be 256-byte aligned");
  }
  const int64_t tokens = batch * seq;
  if (tokens == 0 && !sums) return SWATTN_OK;
  backward_groups(tokens, heads_q, heads_kv, p.groups);
  p.grad[0] = static_cast<const uint16_t*>(grad_q);
  p.grad[1] = static_cast<const uint16_t*>(grad_k);
  p.weight[0] = q_weight;
  p.weight[1] = k_weight;
  p.dx[0] = static_cast<uint16_t*>(dq);
  p.dx[1] = static_cast<uint16_t*>(dk);
  float* ws = static_cast<float*>(workspace);
  if (dq_weight != nullptr) p.part[0] = ws;
  if (dk_weight != nullptr) p.part[1] = ws + static_cast<int64_t>(p.groups[0]) * kD;
  p.heads[0] = heads_q;
  p.heads[1] = heads_kv;
  p.weight_bf16 = weight_bf16;
  p.eps = eps;
  p.seq = static_cast<int>(seq);
  p.tokens = static_cast<int>(tokens);
  p.shares[0] = shares_of(tokens, passes_of(heads_q), p.groups[0]);
  p.shares[1] = shares_of(tokens, passes_of(heads_kv), p.groups[1]);
  const dim3 grid(static_cast<uint32_t>(p.groups[0] + p.groups[1]));
  const int64_t rows = tokens * (int64_t{heads_q} + heads_kv) * (2 * kD);   // bytes of one set of rows
  const int64_t read = tokens * 2 * kD * (heads_q * (q_weight != nullptr ? 2 : 1) + heads_kv * int64_t{k_weight != nullptr ? 2 : 1});
  const bool out = read + rows >= kStreamBytes, in = read >= kCacheBytes;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, as_stream(stream), p); };
  if (interleaved && in)
    launch(rotary_backward_kernel<true, true, true>);
  else if (interleaved && out)
    launch(rotary_backward_kernel<true, false, true>);
  else if (interleaved)
    launch(rotary_backward_kernel<true, false, false>);
  else if (in)
    launch(rotary_backward_kernel<false, true, true>);
  else if (out)
    launch(rotary_backward_kernel<false, false, true>);
  else
    launch(rotary_backward_kernel<false, false, false>);
  if (sums) {
    const SumParams s{{p.part[0], p.part[1]}, {dq_weight, dk_weight}, {p.groups[0], p.groups[1]}, weight_bf16};
    hipLaunchKernelGGL(rotary_sum_kernel, dim3(kD / kSumDims, 2), dim3(256), 0, as_stream(stream), s);
  }
  return launch_status(name);
}

}  // extern "C"
