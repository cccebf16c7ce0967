// What the rotary and the cache kernels share: 16-byte conversions, the rotation
// of two vectors, and the 8-bit rows of the quantised cache.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

namespace bw {

__device__ __forceinline__ void bf16x8_to_f32(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t f32_to_bf16x2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint4 f32_to_bf16x8(const float* x) {
  return make_uint4(f32_to_bf16x2(x[0], x[1]), f32_to_bf16x2(x[2], x[3]), f32_to_bf16x2(x[4], x[5]),
                    f32_to_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ float4 ldg4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }

// The V angles (cos or sin part of a table row) of two vectors of V elements at
// e0 and e1 = e0 + R / 2: pairs (i, i + R/2) share the V angles e0 .., pairs
// (2i, 2i + 1) have V / 2 from e0 / 2 and V / 2 from e1 / 2.
template <int V, bool HALF>
__device__ __forceinline__ void load_angles(const float* row, int e0, int e1, float* x) {
  if constexpr (V == 8) {
    const float4 a = ldg4(row + (HALF ? e0 : e0 / 2)), b = ldg4(row + (HALF ? e0 + 4 : e1 / 2));
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else if constexpr (HALF) {
    const float4 a = ldg4(row + e0);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  } else {
    const float2 a = __ldg(reinterpret_cast<const float2*>(row + e0 / 2));
    const float2 b = __ldg(reinterpret_cast<const float2*>(row + e1 / 2));
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  }
}

// Rotates 2 V elements by V angles: pairs (i, i + V) of the array (HALF) or
// (2i, 2i + 1).  Each product is rounded to fp32 by itself, so that the result
// does not depend on which product a compiler contracts into an FMA: the fused
// write of a rotated K row and the stand-alone rotation agree to the bit.
template <int V, bool HALF>
__device__ __forceinline__ void rotate(float* x, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int ia = HALF ? i : 2 * i, ib = HALF ? i + V : 2 * i + 1;
    const float a = x[ia], b = x[ib];
    x[ia] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    x[ib] = __fadd_rn(__fmul_rn(a, s[i]), __fmul_rn(b, c[i]));
  }
}

// The 8-bit row: codes c = e4m3(x 2^-e), e the smallest integer with
// max|x| <= 448 2^e.  A power of two keeps x 2^-e and c 2^e exact, so a row has
// one rounding (half a step, 2^-4 relative, for elements within 2^14 of the
// row's largest) and reading it back as bf16 adds none.  e is clamped to
// [kMinExp, kMaxExp] and kept as the byte e + 127; a row of zeros has e = 0.
// kMinExp leaves 2^-e and sums over tokens weighted with 2^e inside fp32.
constexpr int kMinExp = -100, kMaxExp = 120;

// `amax`: the largest finite magnitude of the row (>= 0).
__device__ __forceinline__ int row_exponent(float amax) {
  // 448 = 1.75 * 2^8: e = exponent(amax) - 8, one more where the mantissa is above 1.75
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return amax > 0.f ? min(max(e, kMinExp), kMaxExp) : 0;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t f32_to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Four codes -> two half2 (lo: bytes 0 and 1, hi: bytes 2 and 3); every e4m3 value is
// an f16 value.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t four, float* x) {
  uint32_t lo, hi;
  e4m3x4_to_f16x4(four, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

}  // namespace bw
