// Device helpers of the 8-bit KV cache: e4m3 codes with one power-of-two
// scale per block of kKv8Block consecutive slots and KV head, stored as its
// biased exponent (value = code * 2^(exponent - 127)).
//
// Why e4m3 with power-of-two scales: e4m3 is itself a floating-point format,
// so a finer scale buys no precision, only range, and with a power of two
// moving a block to a larger scale and undoing the scale are exact (but for
// codes that become subnormal), so an append that grows a partly filled
// block's scale does not wear its older tokens down, and the attention kernels
// fold the scales into exponents.
#pragma once

#include <stdint.h>

#include "fe_common.cuh"

namespace fe {

constexpr int kKv8Block = 16;  // slots per scale
// Exponents an append writes: 2^-32 .. 2^64. The limits keep every block's
// softmax weight and value scale together inside fp32's exponent range, and
// let a block of zeros have a scale.
constexpr int kKv8MinExp = 95, kKv8MaxExp = 191;

// Two e4m3 codes (low byte first) from two floats, nearest even, saturating
// at +-448; NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes (the low 16 bits of `c`) as a half pair; every e4m3 value is a
// half exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t c) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
      : "=r"(r)
      : "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_h2(uint32_t c) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
      : "=r"(r)
      : "r"(c));
  return r;
}

// 2^(e - 127) of a biased exponent in [1, 254].
__device__ __forceinline__ float exp_scale(int e) { return __int_as_float(e << 23); }
// A stored exponent as the attention kernels use it: the limits of an append,
// so that bytes of blocks no token was written to stay finite.
__device__ __forceinline__ int exp_clamp(int e) { return min(max(e, kKv8MinExp), kKv8MaxExp); }

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Packed 16-bit maximum of magnitudes (a NaN is passed over).
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t v, __half) {
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&m),
                            __habs2(*reinterpret_cast<__half2*>(&v)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t v, __nv_bfloat16) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&m),
                                   __habs2(*reinterpret_cast<__nv_bfloat162*>(&v)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

}  // namespace fe
