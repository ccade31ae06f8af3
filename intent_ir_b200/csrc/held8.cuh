// Values held in 8 bits with an f32 scale: e4m3 (largest 448) or int8 (symmetric, largest 127).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace ib200 {

enum : int { HELD_E4M3 = 1, HELD_I8 = 2 };

#ifdef __CUDACC__
template <int HELD> __device__ __forceinline__ constexpr float held_top() { return HELD == HELD_E4M3 ? 448.0f : 127.0f; }
// 1 / Q in f32: a scale is the largest magnitude times this
template <int HELD> __device__ __forceinline__ constexpr float held_unit() { return HELD == HELD_E4M3 ? 1.0f / 448.0f : 1.0f / 127.0f; }
// What a value is multiplied by before it is rounded: Q / max|y|, 0 for a group of zeros (which then holds zeros) and where the
// quotient overflows (max|y| below 2^-119: the group is held as zeros).  A NaN stays a NaN; an infinite maximum gives 0.
template <int HELD> __device__ __forceinline__ float held_inverse(float top) {
  const float inv = held_top<HELD>() / top;
  return top == 0.0f || isinf(inv) ? 0.0f : inv;
}
template <int HELD> __device__ __forceinline__ uint32_t hold1(float v) {
  if (HELD == HELD_E4M3) return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)(uint8_t)(int8_t)max(-127, min(127, __float2int_rn(v)));  // half to even; NaN gives 0
}
template <int HELD> __device__ __forceinline__ uint32_t hold4(float a, float b, float c, float d) {
  if (HELD == HELD_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  return hold1<HELD>(a) | hold1<HELD>(b) << 8 | hold1<HELD>(c) << 16 | hold1<HELD>(d) << 24;
}
// 8 adjacent values times `inv`; vec: p is 8-byte aligned
template <int HELD> __device__ __forceinline__ void hold8(uint8_t* p, const float (&v)[8], float inv, bool vec, int left) {
  if (vec && left >= 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(hold4<HELD>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                                              hold4<HELD>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (uint8_t)hold1<HELD>(v[i] * inv);
  }
}
template <int HELD> __device__ __forceinline__ float held_value(uint8_t b) {
  if (HELD == HELD_I8) return (float)(int8_t)b;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}
// four bytes as two pairs of f16, exact
template <int HELD> __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (HELD == HELD_E4M3) {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {  // the byte as 1024 + (i + 128), minus 1152
    w ^= 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 a = __hsub2(*reinterpret_cast<__half2*>(&l), off), b = __hsub2(*reinterpret_cast<__half2*>(&h), off);
    lo = *reinterpret_cast<uint32_t*>(&a);
    hi = *reinterpret_cast<uint32_t*>(&b);
  }
}
#endif

}  // namespace ib200
