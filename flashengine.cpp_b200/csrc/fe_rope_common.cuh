// The rotation of two pairs of a head, shared by the rotary kernels
// (fe_rope_accept.cu, fe_rope_axes.cu): every product and sum is rounded to
// fp32 by itself, the result once to the 16-bit type.
#pragma once

#include "fe_common.cuh"

namespace fe {

template <typename T>
struct Pair2;
template <>
struct Pair2<__half> {
  using V = __half2;
  static __device__ __forceinline__ float2 to_float(V x) { return __half22float2(x); }
  static __device__ __forceinline__ V from_float(float a, float b) {
    return __halves2half2(__float2half_rn(a), __float2half_rn(b));
  }
};
template <>
struct Pair2<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static __device__ __forceinline__ float2 to_float(V x) { return __bfloat1622float2(x); }
  static __device__ __forceinline__ V from_float(float a, float b) {
    return __halves2bfloat162(__float2bfloat16_rn(a), __float2bfloat16_rn(b));
  }
};

// Rotate the pairs (j, j+r) and (j+1, j+r+1) of one head in registers (r =
// half the rotary dims), given cos c and sin s of both.
template <typename T>
__device__ __forceinline__ void rotate(typename Pair2<T>::V& lo, typename Pair2<T>::V& hi,
                                       float2 c, float2 s) {
  const float2 a = Pair2<T>::to_float(lo), b = Pair2<T>::to_float(hi);
  lo = Pair2<T>::from_float(__fsub_rn(__fmul_rn(a.x, c.x), __fmul_rn(b.x, s.x)),
                            __fsub_rn(__fmul_rn(a.y, c.y), __fmul_rn(b.y, s.y)));
  hi = Pair2<T>::from_float(__fadd_rn(__fmul_rn(b.x, c.x), __fmul_rn(a.x, s.x)),
                            __fadd_rn(__fmul_rn(b.y, c.y), __fmul_rn(a.y, s.y)));
}

}  // namespace fe
