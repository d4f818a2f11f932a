// Formats of the 8-bit K/V cache.
//
// A pool holds codes [num_slots, Hkv, D] and one fp32 scale per (block, kv
// head); a row's value is code * scale. The scales the cache write makes are
// powers of two: dividing by one is exact, so the only rounding of a value
// written under its block's final scale is the code's own (half a unit of its
// last place: 2^-4 of the value in e4m3, scale / 2 in int8). Raising a scale
// later moves an e4m3 code without another rounding unless it becomes
// subnormal, but rounds an int8 code again: each scale s that it went through
// adds up to s / 2, and every one is at most half of the next, so a value of a
// block whose scale grew is off by less than one unit of the final scale (e4m3:
// 2^-4 of the value and less than 2^-9 of the scale). For a floating-point code
// a finer scale would gain nothing. An int8 one loses up to a bit against
// amax / 127 (the largest code lies between 64 and 127); powers of two are kept
// there too, since a scale then grows by doublings alone, so that not every
// larger row rounds its block's codes again, and code * scale is exact in 16-bit
// rows. Readers multiply by the scale in fp32 and take any value of it.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace irb {

using e4m3_t = __nv_fp8_e4m3;

template <> struct DT<e4m3_t> {
  __device__ static float to_f(e4m3_t x) { return static_cast<float>(x); }
};
template <> struct DT<int8_t> {
  __device__ static float to_f(int8_t x) { return static_cast<float>(x); }
};

// Smallest power of two s >= 2^-126 with amax / s <= the format's largest
// magnitude: 448 = 1.75 * 2^8 (e4m3), 127 = 1.984375 * 2^6 (int8). amax is
// finite and >= 0; its mantissa decides between two neighbouring exponents.
template <typename C>
__device__ __forceinline__ float scale_for(float amax) {
  constexpr bool kInt = std::is_same<C, int8_t>::value;
  constexpr uint32_t kTop = kInt ? 0x7e0000u : 0x600000u;  // mantissa bits of the largest
  constexpr int kExp = kInt ? 6 : 8;
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - kExp + ((u & 0x7fffffu) > kTop ? 1 : 0);  // biased
  e = e < 1 ? 1 : e;
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// 1 / s of a normal power of two s in [2^-126, 2^126], exact; 0 if s is not one.
__device__ __forceinline__ float pow2_reciprocal(float s) {
  const uint32_t u = __float_as_uint(s);
  const uint32_t e = u >> 23;
  return ((u & 0x7fffffu) == 0u && e >= 1u && e <= 253u) ? __uint_as_float((254u - e) << 23)
                                                         : 0.f;
}

// Four fp32 values (already divided by the scale) as four codes, ties to even.
template <typename C> __device__ __forceinline__ uint32_t encode4(float4 v);
template <>
__device__ __forceinline__ uint32_t encode4<e4m3_t>(float4 v) {
  uint16_t lo, hi;  // saturating; infinities are made NaN by the caller
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v.y), "f"(v.x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v.w), "f"(v.z));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
template <>
__device__ __forceinline__ uint32_t encode4<int8_t>(float4 v) {
  auto one = [](float x) {
    const int i = max(min(__float2int_rn(x), 127), -127);  // NaN converts to 0
    return static_cast<uint32_t>(i) & 0xffu;
  };
  return one(v.x) | (one(v.y) << 8) | (one(v.z) << 16) | (one(v.w) << 24);
}

// Four codes of a 32-bit word as two packed fp16 pairs, exactly. e4m3 by the
// conversion instruction; int8 by placing the byte (offset by 128) under the
// exponent of 1024, whose units are 1, and subtracting 1024 + 128.
template <typename C> __device__ __forceinline__ void decode4_h(uint32_t w, uint32_t& lo,
                                                                uint32_t& hi);
template <>
__device__ __forceinline__ void decode4_h<e4m3_t>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
template <>
__device__ __forceinline__ void decode4_h<int8_t>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);
  const uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
  const uint32_t off = 0x64806480u;  // 1152 twice
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(off));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(off));
}

template <typename C>
__device__ __forceinline__ float4 decode4(uint32_t w) {
  uint32_t lo, hi;
  decode4_h<C>(w, lo, hi);
  const float2 a = unpack2<__half>(lo), b = unpack2<__half>(hi);
  return make_float4(a.x, a.y, b.x, b.y);
}

}  // namespace irb
