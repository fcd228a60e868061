// e4m3 codes (sign, 4 exponent bits of bias 7, 3 mantissa bits; 448 is the largest, 0x7f / 0xff are NaN) <-> fp32.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace llmctl {

// Two numbers to two codes (the first in the low byte), rounded to nearest even; beyond 448 they saturate, NaN stays NaN.
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes to two numbers: exact.
__device__ __forceinline__ float2 unpack_e4m3x2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) { return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16); }
__device__ __forceinline__ uint2 pack_e4m3x8(const float (&f)[8]) {
  return make_uint2(pack_e4m3x4(f[0], f[1], f[2], f[3]), pack_e4m3x4(f[4], f[5], f[6], f[7]));
}
__device__ __forceinline__ void unpack_e4m3x4(uint32_t codes, float* f) {
  const float2 a = unpack_e4m3x2(codes), b = unpack_e4m3x2(codes >> 16);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}
__device__ __forceinline__ void unpack_e4m3x8(uint2 codes, float (&f)[8]) {
  unpack_e4m3x4(codes.x, f);
  unpack_e4m3x4(codes.y, f + 4);
}

}  // namespace llmctl
