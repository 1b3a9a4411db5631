// The two 8-bit formats of the block-wise KV cache (kv_cache.cu writes it, cached_attention*.cu read it).
//
// A stored number stands for code * scale with one scale per (block, kv head). Scales are powers of two, 2^e with the
// least e >= kMinExponent that fits the block's largest magnitude: dividing by one is exact, so a number is rounded
// once, to its code, and moving a block to a larger scale shifts the codes it holds (an e4m3 code keeps its bits unless
// it leaves the normal range, an int8 code drops its lowest). With a scale amax / 448 every growth would round all the
// codes again.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"

namespace qw {

enum KvFormat : int { kKvFp8 = 0, kKvInt8 = 1 };

// Scales stop shrinking here: a code's step is then 2^-64 (int8) or at least 2^-73 (e4m3, whose subnormals are multiples of
// 2^-9), and magnitudes up to half of that become zero.
constexpr int kMinExponent = -64;

template <int FMT>
struct Kv;

template <>
struct Kv<kKvFp8> {
  // amax = m * 2^x with m in [0.5, 1): 448 = 0.875 * 2^9
  static constexpr float kTop = 0.875f;
  static constexpr int kUp = 9;

  __device__ static __forceinline__ uint8_t encode(float x) {  // x already divided by the scale; saturates, NaN stays
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  }
  __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  // two pairs of codes (bytes 0, 1 and 2, 3) as f16 pairs; every code is a half-precision number
  __device__ static __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
  // bit 7 of each byte whose code is a NaN (0x7f, 0xff)
  __device__ static __forceinline__ uint32_t nan_bytes(uint32_t w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  }
};

template <>
struct Kv<kKvInt8> {
  static constexpr float kTop = 0.9921875f;  // 127 = 0.9921875 * 2^7
  static constexpr int kUp = 7;

  __device__ static __forceinline__ uint8_t encode(float x) {  // saturates; NaN becomes 0 (int8 has none)
    const int i = x == x ? __float2int_rn(fminf(fmaxf(x, -127.f), 127.f)) : 0;
    return static_cast<uint8_t>(i);
  }
  __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    return static_cast<uint32_t>(encode(a)) | (static_cast<uint32_t>(encode(b)) << 8) |
           (static_cast<uint32_t>(encode(c)) << 16) | (static_cast<uint32_t>(encode(d)) << 24);
  }
  // code + 128 in the low mantissa byte of 1024.0 (0x6400), minus 1152: exact in half precision
  __device__ static __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
  __device__ static __forceinline__ uint32_t nan_bytes(uint32_t) { return 0; }
};

// The least e >= kMinExponent with amax <= largest code * 2^e (amax finite and not negative).
template <int FMT>
__device__ __forceinline__ int scale_exponent(float amax) {
  if (!(amax > 0.f)) return kMinExponent;
  int x;
  const float m = frexpf(amax, &x);
  return max(kMinExponent, x - Kv<FMT>::kUp + (m > Kv<FMT>::kTop ? 1 : 0));
}

// 2^e for e in [-126, 127]
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

}  // namespace qw
