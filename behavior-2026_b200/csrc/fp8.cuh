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

// Sixteen values as they lie in memory.  Magnitudes are compared as bit patterns of bf16 or fp32 (infinities and NaNs are
// above all finite ones).  These kernels are bound by instruction issue before memory, so the work on a value is
// kept to about five instructions.
template <typename X>
struct Fp8Raw;
template <>
struct Fp8Raw<bf16> {
  uint32_t w[8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const bf16* p) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  }
  __device__ __forceinline__ void load_some(const bf16* p, int n) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) w[i / 2] |= (uint32_t)h[i] << (16 * (i & 1));
  }
  __device__ __forceinline__ uint32_t top() const {  // the largest magnitude's bf16 pattern (any NaN: 0x7fff)
    auto m2 = [](uint32_t a, uint32_t b) {
      const __nv_bfloat162 r = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
      return *reinterpret_cast<const uint32_t*>(&r);
    };
    const uint32_t m = m2(m2(m2(w[0], w[1]), m2(w[2], w[3])), m2(m2(w[4], w[5]), m2(w[6], w[7])));
    return max(m >> 16, m & 0xffffu);
  }
  // the scale byte of a largest magnitude 1.m * 2^x: x - 8 + 127, one more where 1.m > 1.75 (448 = 1.75 * 2^8)
  static constexpr uint32_t BAD = 0x7f80u;
  __device__ __forceinline__ static int byte(uint32_t top) { return max((int)((top + 0x1fu) >> 7) - 8, 0); }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
};
template <>
struct Fp8Raw<float> {
  uint32_t w[16];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 a = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
    }
  }
  __device__ __forceinline__ void load_some(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) w[i] = __float_as_uint(p[i]);
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
  static constexpr uint32_t BAD = 0x7f800000u;
  __device__ __forceinline__ static int byte(uint32_t top) { return max((int)((top + 0x1fffffu) >> 23) - 8, 0); }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
};

// The codes of a lane's sixteen values and the exponent byte of the block that LANES consecutive lanes hold.
// Every lane of the warp calls it.
template <int LANES, typename X>
__device__ __forceinline__ uint4 fp8_encode16(const Fp8Raw<X>& x, int& byte) {
  uint32_t m = x.top();
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const bool bad = m >= Fp8Raw<X>::BAD;  // an infinity or a NaN: codes 0
  const int b = Fp8Raw<X>::byte(m);      // at most 247
  byte = bad ? 255 : b;
  const float r = __uint_as_float((uint32_t)(254 - b) << 23);
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = fp8_pack4(x.at(4 * i) * r, x.at(4 * i + 1) * r, x.at(4 * i + 2) * r, x.at(4 * i + 3) * r);
  return bad ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(c[0], c[1], c[2], c[3]);
}

}  // namespace p5
