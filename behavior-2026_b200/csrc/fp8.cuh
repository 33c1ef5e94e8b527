// fp8.cuh — the 8-bit storage format of the pi05_fp8_* and pi05_kv8_* operators.
//
// A block of values (128 along a row of a GEMM operand, one head of one cached position) is stored as
// e4m3 codes c_i and one exponent byte s: x_i ~ c_i * 2^(s - 127).  s - 127 is the smallest e with
// max|x| <= 448 * 2^e, so scaling is exact and the only rounding is the one to e4m3 (at most 2^-4 of the value,
// or 2^-10 of the scale below the smallest normal code).  A power of two instead of max / 448 costs
// at most the lowest binade of the codes' range and keeps every later product with the scale exact; it is
// also what the tensor cores apply by themselves (kind::mxf8f6f4).
// A block of zeros has s = 0; a block that holds a NaN or an infinity has s = 255 and codes 0, and every
// value of it reads as NaN.
#pragma once
#include "common.cuh"

namespace p5 {

constexpr int FP8_BLOCK = 128;

// exponent byte of a block whose largest finite magnitude is `amax` (>= 0, finite)
__device__ __forceinline__ int fp8_scale_byte(float amax) {
  if (amax == 0.f) return 0;
  const uint32_t u = __float_as_uint(amax);
  // amax = 1.m * 2^x; amax <= 448 * 2^e = 1.75 * 2^(8 + e)  <=>  e >= x - 8 (1.m <= 1.75) or x - 7
  int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased by 127 like the byte itself
  return min(max(e, 0), 254);  // subnormal amax: its own exponent field is 0, so the byte stays 0
}
// 2^(b - 127) for b in [0, 254]; NaN for 255
__device__ __forceinline__ float fp8_scale_value(int b) {
  const uint32_t u = b == 0 ? 0x400000u : (b == 255 ? 0x7fc00000u : (uint32_t)b << 23);
  return __uint_as_float(u);
}
// 2^(127 - b) for b in [0, 254]
__device__ __forceinline__ float fp8_scale_inverse(int b) {
  return __uint_as_float(b == 254 ? 0x400000u : (uint32_t)(254 - b) << 23);
}
// four e4m3 codes (round to nearest even; finite inputs within +-448 after scaling)
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// two codes (low byte first) -> two fp16, exact
__device__ __forceinline__ uint32_t fp8_to_h2(uint16_t c2) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c2));
  return r;
}
__device__ __forceinline__ float2 fp8_to_f2(uint16_t c2) {
  const uint32_t h = fp8_to_h2(c2);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Exponent byte of the block that LANES consecutive lanes hold 8 values of each (0 where a lane has none), and
// the lane's 8 codes.  Every lane of the warp calls it.
template <int LANES>
__device__ __forceinline__ uint2 fp8_encode8(const float (&f)[8], int& byte) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));  // fmaxf drops a NaN: counted below
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= !(fabsf(f[i]) <= 3.4028234e38f);
  if (bad) m = INFINITY;
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m == INFINITY) {
    byte = 255;
    return make_uint2(0u, 0u);
  }
  byte = fp8_scale_byte(m);
  const float r = fp8_scale_inverse(byte);
  return make_uint2(fp8_pack4(f[0] * r, f[1] * r, f[2] * r, f[3] * r), fp8_pack4(f[4] * r, f[5] * r, f[6] * r, f[7] * r));
}

}  // namespace p5
