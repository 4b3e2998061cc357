// Codes and scales of the 8-bit KV cache (include/swattn_cache.h).
#pragma once

#include "common.h"
#include "swattn_cache.h"

namespace swattn {
namespace code {

constexpr int kE4m3 = SWATTN_CODE_E4M3, kInt8 = SWATTN_CODE_INT8;
constexpr int kMinExp = -100;   // scales stay normal numbers, and so do their reciprocals

// 16 codes (one 16-byte piece of a row) as fp32.
template <int kCode>
__device__ __forceinline__ void decode4(uint32_t w, float* x) {
  if constexpr (kCode == kE4m3) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 3);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
}
template <int kCode>
__device__ __forceinline__ void decode16(const uint4& u, float (&x)[16]) {
  decode4<kCode>(u.x, x);
  decode4<kCode>(u.y, x + 4);
  decode4<kCode>(u.z, x + 8);
  decode4<kCode>(u.w, x + 12);
}

// fp32 values inside the codes' range to codes, to nearest, ties to even; NaN to
// the NaN code, or 0 where there is none.
template <int kCode>
__device__ __forceinline__ uint32_t encode4(const float* x) {
  if constexpr (kCode == kE4m3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true));
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = __builtin_rintf(x[i]);
      w |= (static_cast<uint32_t>(static_cast<int>(r == r ? r : 0.f)) & 0xffu) << (8 * i);
    }
    return w;
  }
}
template <int kCode>
__device__ __forceinline__ uint4 encode16(const float (&x)[16]) {
  return make_uint4(encode4<kCode>(x), encode4<kCode>(x + 4), encode4<kCode>(x + 8), encode4<kCode>(x + 12));
}

// The smallest power of two >= 2^kMinExp with |x| <= qmax * scale, from the bits
// of the largest |x| (bits order like magnitudes, infinities and NaN above all);
// NaN for an infinity or a NaN.  qmax = (1 + m) * 2^e: the exponent of |x| less
// e, one more where its mantissa exceeds m.
template <int kCode>
__device__ __forceinline__ float scale_for(uint32_t amax_bits) {
  constexpr int kQmaxExp = kCode == kE4m3 ? 8 : 6;                          // 448 = 1.75 * 2^8
  constexpr uint32_t kQmaxMant = kCode == kE4m3 ? 0x600000u : 0x7e0000u;    // 127 = 1.984375 * 2^6
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  int e = static_cast<int>(amax_bits >> 23) - 127 - kQmaxExp + ((amax_bits & 0x7fffffu) > kQmaxMant ? 1 : 0);
  e = e < kMinExp ? kMinExp : e;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Scaled values of a block with this scale, cut to the largest code whose value bf16
// still holds.  Only the largest numbers need it: above 240 * 2^120 (e4m3) and 63 * 2^122
// (int8) the nearest code would stand for 2^128.
template <int kCode>
__device__ __forceinline__ void keep_finite(float scale, float (&x)[16]) {
  constexpr float kMax = 0x1.fep127f, kQmax = kCode == kE4m3 ? 448.f : 127.f;
  if (scale > kMax / kQmax) {
    float top = kMax / scale;   // to the code below it
    top = kCode == kE4m3 ? __uint_as_float(__float_as_uint(top) & 0xfff00000u) : __builtin_truncf(top);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = x[j] > top ? top : x[j] < -top ? -top : x[j];   // NaN stays NaN
  }
}

// T's bytes at `at`, loaded as Raw; kStream: past the memory-side cache (data that is
// there all the same is read from it).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool kStream, class Raw, class T>
__device__ __forceinline__ T load_bytes(const uint8_t* at) {
  const Raw* p = reinterpret_cast<const Raw*>(at);
  if constexpr (kStream) return __builtin_bit_cast(T, __builtin_nontemporal_load(p));
  return __builtin_bit_cast(T, *p);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Host: the blocks that there are kernels for.
inline bool block_ok(int32_t block) { return block == 16 || block == 32 || block == 64 || block == 128; }

}  // namespace code
}  // namespace swattn
