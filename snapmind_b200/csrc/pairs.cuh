// Small arithmetic that the chunk kernels and the 8-bit pool share: pairs of f32, pairs of 16-bit elements,
// e4m3 codes and their scale bytes.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace snapmind {

constexpr float kLog2e = 1.4426950408889634f;

// Pairs of f32 in one instruction: a b + c, a + b, a times one factor.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 x, x, y, z; "
      "mov.b64 {%0, %1}, x; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 times(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float b) {
  float2 r;
  asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %4}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b));
  return r;
}

// Two f32 rounded to a word of two 16-bit elements.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// e4m3 codes as f16 (exact): four to two words (the low two codes, the high two); one to f32.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float e4m3_to_f(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }
// 2^(b - 127) of a scale byte in [27, 247] (a normal float's exponent field).
__device__ __forceinline__ float scale_byte_to_f(uint32_t b) { return __uint_as_float(b << 23); }

// e4m3 rows: the exponent of a row whose largest finite magnitude is a.
__device__ __forceinline__ int row_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int k = (int)(u >> 23) - 127;
  const int e = (u & 0x7FFFFFu) <= 0x600000u ? k - 8 : k - 7;  // a <= 1.75 2^(e + 8)
  return min(max(e, -100), 120);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // false for NaN too
}
__device__ __forceinline__ float scaled(float x, float inv) {
  return fabsf(x) < INFINITY ? x * inv : __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t codes2(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) { return codes2(a, b) | (codes2(c, d) << 16); }

}  // namespace snapmind
