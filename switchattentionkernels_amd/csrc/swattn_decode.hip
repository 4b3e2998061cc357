// Routed GQA decode for gfx950: one new query token per sequence attends its
// KV cache, either fully (causal over the whole cache) or over the last
// `window` keys -- the routing rule of the prefill path applied to its last
// row (F:145-155: query position p = len - 1 sees keys [0, p] when full and
// [p - window + 1, p] when local).  The reference has no decode path.
//
// HBM-bound: every cached key and value of the routed range is read once per
// KV head.  Split-K: the routed keys of all (sequence, KV head) pairs, pair
// after pair, form one line, and every workgroup streams an equal share of it
// with an online softmax, so that one long sequence, many short ones and any
// mix of full and local sequences load the chip evenly in a single round of
// workgroups.  Which keys are routed is known only on the device: up to
// kInlineSeqs sequences every workgroup finds its share by itself
// (plan_inline); beyond that a one-workgroup kernel writes the sequences'
// places on the line first.  A last kernel merges the fp32 partials in the
// log2 domain (LSE as V:236-241).
//
// Layout: q [B, Hq, 128], caches [B, L, Hkv, 128] bf16; out [B, Hq, 128] bf16,
// lse [B, Hq] fp32.  Group size G = Hq / Hkv <= 8.

#include <mutex>
#include <string>

#include "decode_line.h"

namespace swattn {
namespace {

constexpr int kDecWaves = 4;         // waves per workgroup
constexpr int kMaxG = 8;
constexpr uint32_t kPairPad = 192;   // a pair's start, in keys

struct DecodeParams : DecodeCommon {
  static constexpr uint32_t kMinShare = 128;     // line positions per workgroup, at least (64 and
                                                 // 256: up to 7 % and 10 % slower on single short caches)
  static constexpr uint32_t kLongShare = 2048;   // shares from this length on are halved
  static constexpr uint32_t kAlignSlack = 80;
  static constexpr bool kKeepNan = false;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  float c;           // sm_scale * log2(e)
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

// Streams K and V at 5.2 TB/s where sequences are long (B64 L4096-8192 all
// full, whole call 345 -> 310 us against chunks planned by a kernel of their
// own with up to three uneven rounds of workgroups); B64 p_full 0.25 152 ->
// 139 us, B24 L1500-3000 p_full 0.5 60 -> 44 us, B1 L2048-4096 22.8 -> 14.6 us.
// Short calls are bound by their dependent latencies: plan, Q and first keys,
// the combine, and the merge kernel's launch.
//
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
template <int G, bool kInline>
__global__ __launch_bounds__(256) void decode_split_kernel(const DecodeParams p) {
  __shared__ float s_m[kDecWaves][G], s_l[kDecWaves][G];
  __shared__ float s_acc[kDecWaves][G][kD];
  __shared__ SeqEntry s_ent[kInline ? kInlineSeqs : 1];
  SplitStart st;
  if constexpr (kInline) {
    if (!plan_inline(p, s_ent, st)) return;
  } else {
    if (!plan_listed(p, st)) return;
  }
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
    const int64_t slot = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(r) * p.hkv + kvh;
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
        const uint32_t vx[4] = {vr[j].x, vr[j].y, vr[j].z, vr[j].w};
#pragma unroll
        for (int h = 0; h < G; ++h) {
          const float pr = live ? __builtin_amdgcn_exp2f(s[h] - m[h]) : 0.f;
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
      const float a = mm == -INFINITY ? 0.f : exp2f(m[h] - mm);
      float lh = l[h] * a;
      lh += __shfl_xor(lh, 16);
      lh += __shfl_xor(lh, 32);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        float x = acc[h][d] * a;
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        if (kg == 0) s_acc[wave][h][8 * ds + d] = x;
      }
      if (lane == 0) {
        s_m[wave][h] = mm;
        s_l[wave][h] = lh;
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
      for (int w = 0; w < kDecWaves; ++w) mm = fmaxf(mm, s_m[w][h]);
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w)
        if (s_m[w][h] != -INFINITY) a += exp2f(s_m[w][h] - mm) * s_acc[w][h][d];
      po[i] = a;
    }
    if (tid < G) {
      float mm = -INFINITY, lh = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) mm = fmaxf(mm, s_m[w][tid]);
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w)
        if (s_m[w][tid] != -INFINITY) lh += exp2f(s_m[w][tid] - mm) * s_l[w][tid];
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

__global__ __launch_bounds__(256) void decode_merge_kernel(const DecodeParams p) { merge_row(p, blockIdx.x); }

}  // namespace
}  // namespace swattn

using namespace swattn;

extern "C" {

// Workgroups the line of routed keys is shared out over: two per CU, as many
// as are resident at once for the larger query groups.  The workspace holds
// four per CU plus one per (sequence, KV head) pair partials; shares number
// at most that many and each pair adds at most one piece.
constexpr int kSplitTarget = 2;   // workgroups per CU
constexpr int kSplitRoom = 4;     // partials per CU in the workspace
static_assert(2 * kSplitTarget <= kSplitRoom, "every share has its partial");

static int decode_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    return 256;
  return n;
}

struct DecodeLayout {
  int64_t slots, off_ml, off_list, off_plan, bytes;   // byte offsets
};

static DecodeLayout decode_layout(int64_t batch, int64_t heads_q, int64_t heads_kv, int cus) {
  DecodeLayout L{};
  L.slots = static_cast<int64_t>(kSplitRoom) * cus + batch * heads_kv;
  const int64_t group = heads_q / heads_kv;
  auto al = [](int64_t x) { return (x + 255) & ~static_cast<int64_t>(255); };
  int64_t o = al(L.slots * group * kD * 4);               // part_o
  L.off_ml = o;    o = al(o + L.slots * group * 2 * 4);
  L.off_list = o;  o = al(o + batch * 4);
  L.off_plan = o;  o = al(o + (1 + batch) * 16);
  L.bytes = o;
  return L;
}

size_t swattn_decode_workspace_bytes(int32_t batch, int64_t cache_len, int32_t heads_q,
                                     int32_t heads_kv) {
  if (batch < 1 || cache_len < 1 || heads_q < 1 || heads_kv < 1 || heads_q % heads_kv) return 0;
  return static_cast<size_t>(decode_layout(batch, heads_q, heads_kv, decode_cus()).bytes);
}

}  // extern "C"

// Argument checks shared by both decode entry points (name = the entry point).
static int decode_check(const char* name, const void* q, const void* k_cache,
                        const void* v_cache, const int32_t* cache_lens, const uint8_t* full,
                        void* out, float* lse, int32_t batch, int64_t cache_len,
                        int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t window) {
  const std::string n(name);
  if (head_dim != kD) return invalid(n + ": head_dim must be 128");
  if (batch < 1 || cache_len < 1 || heads_q < 1 || heads_kv < 1) return invalid(n + ": bad shape");
  if (heads_q % heads_kv) return invalid(n + ": heads_q must be a multiple of heads_kv");
  if (heads_q / heads_kv > kMaxG) return invalid(n + ": heads_q / heads_kv must be at most 8");
  if (window <= 0) return invalid(n + ": window must be positive");
  if (batch > 65535 || heads_kv > 65535 || cache_len > INT32_MAX ||
      static_cast<int64_t>(batch) * heads_q > INT32_MAX)
    return invalid(n + ": batch, heads_kv or cache_len too large");
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || cache_lens == nullptr ||
      full == nullptr || out == nullptr || lse == nullptr)
    return invalid(n + ": null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return invalid(n + ": q, k_cache, v_cache and out must be 16-byte aligned");
  return SWATTN_OK;
}

template <int G>
static void launch_split(bool inline_plan, dim3 grid, hipStream_t st, const DecodeParams& p) {
  if (inline_plan)
    hipLaunchKernelGGL((decode_split_kernel<G, true>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((decode_split_kernel<G, false>), grid, dim3(256), 0, st, p);
}

// Split and merge kernels (and the plan kernel for many sequences) on `stream`
// with the (checked) workspace ws.
static int decode_launch(const char* name, const void* q, const void* k_cache,
                         const void* v_cache, const int32_t* cache_lens, const uint8_t* full,
                         void* out, float* lse, int32_t batch, int64_t cache_len,
                         int32_t heads_q, int32_t heads_kv, int32_t window, float scale_log2,
                         char* ws, void* stream) {
  const int group = heads_q / heads_kv;
  DecodeParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k_cache);
  p.v = static_cast<const uint16_t*>(v_cache);
  p.lens = cache_lens;
  p.full = full;
  const int cus = decode_cus();
  const DecodeLayout L = decode_layout(batch, heads_q, heads_kv, cus);
  if (L.slots > INT32_MAX) return invalid(std::string(name) + ": too many work items");
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + L.off_ml);
  p.list = reinterpret_cast<int32_t*>(ws + L.off_list);
  p.plan = reinterpret_cast<uint4*>(ws + L.off_plan);
  p.target = kSplitTarget * cus;
  // A share is at most the line over the resident workgroups, and has to fit 32
  // bits: with 256 CUs the limit is 128 TiB of K, the size of the address space.
  const int64_t rows = static_cast<int64_t>(batch) * cache_len * heads_kv;
  if (rows / p.target >= (int64_t{1} << 30))
    return invalid(std::string(name) + ": the K cache is larger than the address space");
  // (Padding positions of the line stay below 2^30 beside at most 2^31 keys.)
  p.pad = static_cast<int64_t>(batch) * heads_kv < (int64_t{1} << 30) / kPairPad ? kPairPad : 0;
  p.batch = batch;
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.cache_len = static_cast<int>(cache_len);
  p.hq = heads_q;
  p.hkv = heads_kv;
  p.group = group;
  p.window = window;
  p.c = scale_log2;
  const hipStream_t st = as_stream(stream);
  // Up to kInlineSeqs sequences the split workgroups plan for themselves, at
  // up to kInlinePer sequences per thread; beyond that each of them would
  // read too many lengths and the plan kernel's few us no longer count
  // beside the thousands of pairs.  (Caches of 2^31 rows, which only a sparsely
  // mapped address range can hold, need the plan kernel's 64-bit positions.)
  const bool inline_plan = batch <= kInlineSeqs && rows <= INT32_MAX;
  if (!inline_plan) hipLaunchKernelGGL(decode_plan_kernel<DecodeParams>, dim3(1), dim3(kPlanThreads), 0, st, p);
  // Grid: one workgroup per share, no more of them than whole caches can fill
  // at kMinShare positions each.
  const int64_t pairs = static_cast<int64_t>(batch) * heads_kv;
  const int64_t most = pairs * ((cache_len + p.pad + DecodeParams::kMinShare - 1) / DecodeParams::kMinShare);
  const dim3 grid(static_cast<uint32_t>(most < 2 * p.target ? most : 2 * p.target));
  switch (group) {
    case 1: launch_split<1>(inline_plan, grid, st, p); break;
    case 2: launch_split<2>(inline_plan, grid, st, p); break;
    case 3: launch_split<3>(inline_plan, grid, st, p); break;
    case 4: launch_split<4>(inline_plan, grid, st, p); break;
    case 5: launch_split<5>(inline_plan, grid, st, p); break;
    case 6: launch_split<6>(inline_plan, grid, st, p); break;
    case 7: launch_split<7>(inline_plan, grid, st, p); break;
    default: launch_split<8>(inline_plan, grid, st, p); break;
  }
  const int64_t out_rows = static_cast<int64_t>(batch) * heads_q;
  hipLaunchKernelGGL(decode_merge_kernel, dim3(static_cast<uint32_t>(out_rows)), dim3(256), 0, st, p);
  return launch_status(name);
}

extern "C" {

int swattn_decode_fwd(const void* q, const void* k_cache, const void* v_cache,
                      const int32_t* cache_lens, const uint8_t* full, void* out, float* lse,
                      int32_t batch, int64_t cache_len, int32_t heads_q, int32_t heads_kv,
                      int32_t head_dim, int32_t window, float scale_log2, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const char* name = "swattn_decode_fwd";
  const int st = decode_check(name, q, k_cache, v_cache, cache_lens, full, out, lse, batch,
                              cache_len, heads_q, heads_kv, head_dim, window);
  if (st != SWATTN_OK) return st;
  const size_t need = swattn_decode_workspace_bytes(batch, cache_len, heads_q, heads_kv);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("swattn_decode_fwd: workspace smaller than swattn_decode_workspace_bytes()");
    return SWATTN_EWORKSPACE;
  }
  if (!aligned256(workspace)) return invalid("swattn_decode_fwd: workspace must be 256-byte aligned");
  return decode_launch(name, q, k_cache, v_cache, cache_lens, full, out, lse, batch, cache_len,
                       heads_q, heads_kv, window, scale_log2, static_cast<char*>(workspace),
                       stream);
}

}  // extern "C"

// ---------------------------------------------------------------------------
// The same decode with library-owned scratch, for callers that cannot
// allocate device memory (code under HIP graph capture, tight serving loops).
// `scratch` is a file-scope device array: every GPU the library runs on gets
// its own copy, held until the process ends.  In host code its name is only a
// host-side stand-in, so its device address is looked up once per device
// (hipGetSymbolAddress, with that device current) and only that address is
// ever handed to kernels.  The decode kernels write every scratch byte they
// read within the same call (plan, list of sequences, partials), so nothing
// needs clearing between calls; two calls that overlap on one GPU share the
// array and race.
// ---------------------------------------------------------------------------
constexpr size_t kDecodeScratchBytes = SWATTN_DECODE_NOALLOC_MAX_BYTES;   // 16 MiB per GPU
static_assert(kDecodeScratchBytes % 256 == 0, "whole 256-byte lines");
static __device__ __align__(256) char scratch[kDecodeScratchBytes];

constexpr int kMaxScratchDevices = 64;
static std::mutex g_scratch_mu;
static void* g_scratch_ptr[kMaxScratchDevices];   // per device, nullptr until looked up

// Device address of this GPU's scratch array (the current device's), or
// nullptr with the error set.
static void* scratch_for_current_device(const char* name) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxScratchDevices) {
    set_error(std::string(name) + ": no usable current device");
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch_ptr[dev] == nullptr) {
    void* ptr = nullptr;
    const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess || ptr == nullptr) {
      set_error(std::string(name) + ": hipGetSymbolAddress(scratch): " + hipGetErrorString(e));
      return nullptr;
    }
    g_scratch_ptr[dev] = ptr;
  }
  return g_scratch_ptr[dev];
}

extern "C" {

int swattn_decode_fwd_noalloc(const void* q, const void* k_cache, const void* v_cache,
                              const int32_t* cache_lens, const uint8_t* full, void* out,
                              float* lse, int32_t batch, int64_t cache_len, int32_t heads_q,
                              int32_t heads_kv, int32_t head_dim, int32_t window,
                              float scale_log2, void* stream) {
  const char* name = "swattn_decode_fwd_noalloc";
  const int st = decode_check(name, q, k_cache, v_cache, cache_lens, full, out, lse, batch,
                              cache_len, heads_q, heads_kv, head_dim, window);
  if (st != SWATTN_OK) return st;
  const size_t need = swattn_decode_workspace_bytes(batch, cache_len, heads_q, heads_kv);
  if (need > kDecodeScratchBytes) {
    set_error("swattn_decode_fwd_noalloc: this shape needs " + std::to_string(need) +
              " bytes of scratch, more than the library's " +
              std::to_string(kDecodeScratchBytes) + " (use swattn_decode_fwd with a workspace)");
    return SWATTN_EINVAL;
  }
  void* ws = scratch_for_current_device(name);
  if (ws == nullptr) return SWATTN_EINVAL;
  return decode_launch(name, q, k_cache, v_cache, cache_lens, full, out, lse, batch, cache_len,
                       heads_q, heads_kv, window, scale_log2, static_cast<char*>(ws), stream);
}

}  // extern "C"
