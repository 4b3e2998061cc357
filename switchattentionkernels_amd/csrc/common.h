// Shared host/device helpers for libswattn.so (gfx950 only).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "swattn.h"

namespace swattn {

// Per-thread message for the last failing C-ABI call.
void set_error(const std::string& msg);

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

// Returns a C-ABI status for the last launch on this thread.
inline int launch_status(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return SWATTN_OK;
}

inline int invalid(const std::string& msg) {
  set_error(msg);
  return SWATTN_EINVAL;
}

// bf16 row tensors (Q, K, V, O and their gradients, caches, partials) move
// in 16-byte pieces, by vector loads and global -> LDS DMAs: their base
// pointers must be 16-byte aligned.
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Workspaces hold float4 / int64 records at 256-byte-aligned offsets from
// their start, which must itself be 256-byte aligned (as hipMalloc returns).
inline bool aligned256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }

// popcount(mask & lanes_below_me) without a lane-mask table.
__device__ __forceinline__ int count_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

__device__ __forceinline__ uint64_t wave_ballot(bool p) { return __builtin_amdgcn_ballot_w64(p); }

// Inclusive sums over the lanes of a wave: shifts within 16 lanes, then the last
// lane of each row of 16 to the rows behind it.
__device__ __forceinline__ uint32_t wave_sums(uint32_t x) {
  int v = static_cast<int>(x);
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return static_cast<uint32_t>(v);
}

// x of a lane that a move within 16 lanes names (DPP control kMove).
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kTurn4 = 0x124, kTurn8 = 0x128;
template <int kMove>
__device__ __forceinline__ float lane_move(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kMove, 0xf, 0xf, false));
}
// op(x, x of lane ^ 32) and of lane ^ 16, for a commutative op.
template <class Op>
__device__ __forceinline__ float with_lane32(float x, Op op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <class Op>
__device__ __forceinline__ float with_lane16(float x, Op op) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// A commutative op over the wave, the same in every lane, as a butterfly over lane
// distances 32, 16, 8, 4, 2, 1 without LDS round trips (after distance 8, x repeats
// every 8 lanes: a turn by 4 is distance 4).
template <class Op>
__device__ __forceinline__ float wave_all(float x, Op op) {
  x = with_lane16(with_lane32(x, op), op);
  x = op(x, lane_move<kTurn8>(x));
  x = op(x, lane_move<kTurn4>(x));
  x = op(x, lane_move<kXor2>(x));
  return op(x, lane_move<kXor1>(x));
}
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

}  // namespace swattn
