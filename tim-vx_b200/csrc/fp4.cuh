// Conversions of 4-bit block floating point: e2m1 codes, e8m0 and e4m3 scales.
#ifndef B2VX_FP4_CUH_
#define B2VX_FP4_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "b2vx.h"

namespace b2vx {

// Eight floats to e2m1 codes (nearest even, cut to +-6), element i in bits 4 i.
__device__ __forceinline__ uint32_t e2m1_codes(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// The values of eight codes.
__device__ __forceinline__ void e2m1_values(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// a and b to e4m3 bytes (nearest even, cut to 448), a in the low byte.
__device__ __forceinline__ uint32_t e4m3_bytes(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(byte)));
  return __half2float(__ushort_as_half(static_cast<uint16_t>(h & 0xffff)));
}
// 2^(b - 127); 255 is NaN.  2^-127 is a subnormal float.
__device__ __forceinline__ float e8m0_value(uint32_t b) {
  return b == 255u ? __int_as_float(0x7fc00000) : (b == 0u ? __int_as_float(0x00400000) : __int_as_float(b << 23));
}
template <int FORMAT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return FORMAT == B2VX_FP4_BLOCK32 ? e8m0_value(byte) : e4m3_value(byte);
}

// e2m1 magnitudes in halves: code c stands for half_units(c) / 2.
__device__ __forceinline__ float e2m1_magnitude(uint32_t c) {
  return c < 2 ? 0.5f * c : __int_as_float((((c >> 1) + 126u) << 23) | ((c & 1u) << 22));
}

// The block's scale byte and the codes of this lane's eight numbers, which are `LANES` lanes' share of a block.
template <int FORMAT>
__device__ __forceinline__ uint32_t quantize_8(float (&v)[8], float g, uint32_t& byte) {
  constexpr int LANES = FORMAT == B2VX_FP4_BLOCK32 ? 4 : 2;
  // magnitudes as integers: NaN is above infinity is above everything else
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  float w[8];
  if (FORMAT == B2VX_FP4_BLOCK32) {
    if (top >= 0x7f800000u) {
      byte = 255u;
      return 0u;
    }
    const int e = static_cast<int>(top >> 23) - 2;       // biased exponent of 2^(floor(log2 amax) - 2)
    byte = static_cast<uint32_t>(max(e, 0));
    const float inv = __uint_as_float((254u - byte) << 23);   // a power of two: products below are exact
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = v[i] * inv;
    return e2m1_codes(w);
  }
  if (top >= 0x7f800000u || !(g > 0.0f) || !(g < __int_as_float(0x7f800000))) {
    byte = 127u;
    return 0u;
  }
  // Tensor scales near the ends of float's range: numbers and scale times one power of two, so that nothing below overflows or loses bits.
  if (g < 0x1p-60f || g > 0x1p60f) {
    const float lift = g < 1.0f ? 0x1p64f : 0x1p-64f;
    g *= lift;
    top = __float_as_uint(__uint_as_float(top) * lift);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= lift;
  }
  // amax / (6 g) in two roundings is off by less than 2^-22 of itself: where a little less and a little more round to the
  // same byte, that is the answer; else the border between them decides, by an exact comparison: border * 6 has few bits and the
  // fused product with g is rounded only after the subtraction.
  const float amax = __uint_as_float(top);
  const float q = amax / (6.0f * g);
  const uint32_t two = e4m3_bytes(q * (1.0f - 0x1p-21f), q * (1.0f + 0x1p-21f));
  byte = two >> 8;
  if ((two & 0xff) != byte) {
    const float border6 = 3.0f * (e4m3_value(two & 0xff) + e4m3_value(byte));
    const float r = fmaf(border6, g, -amax);
    if (r > 0.0f || (r == 0.0f && (byte & 1u))) byte = two & 0xff;
  }
  const float s = e4m3_value(byte);
  if (byte == 0) return 0u;
  // The numbers over s g, by the same argument.
  const float inv = 1.0f / (s * g);
  float hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = v[i] * inv;
    w[i] = y * (1.0f - 0x1p-21f);
    hi[i] = y * (1.0f + 0x1p-21f);
  }
  uint32_t codes = e2m1_codes(w);
  const uint32_t up = e2m1_codes(hi);
  if (codes != up) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = (codes >> (4 * i)) & 7u, b = (up >> (4 * i)) & 7u;
      if (a != b) {
        const float border = 0.5f * (e2m1_magnitude(a) + e2m1_magnitude(b)) * s;
        const float r = fmaf(border, g, -fabsf(v[i]));
        if (r < 0.0f || (r == 0.0f && (a & 1u))) codes += (b - a) << (4 * i);
      }
    }
  }
  return codes;
}

}  // namespace b2vx
#endif  // B2VX_FP4_CUH_
