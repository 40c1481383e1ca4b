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
__device__ __forceinline__ void e2m1_values(uint32_t codes, float* v) {
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

// What quantization needs of block16's tensor scale, worked out once by a thread.
struct TensorScale {
  float g = 1.0f;          // times lift
  float lift = 1.0f;       // numbers are multiplied by it: near the ends of float's range nothing then overflows or loses bits
  float over_g = 1.0f;     // 1 / g
  float over_6g = 1.0f;    // 1 / (6 g)
  bool ok = true;
};
template <int FORMAT>
__device__ __forceinline__ TensorScale tensor_scale(const float* p) {
  TensorScale t;
  if (FORMAT == B2VX_FP4_BLOCK16) {
    const float g = __ldg(p);
    t.ok = g > 0.0f && g < __int_as_float(0x7f800000);
    t.lift = g < 0x1p-60f ? 0x1p64f : (g > 0x1p60f ? 0x1p-64f : 1.0f);
    t.g = g * t.lift;
    t.over_g = 1.0f / t.g;
    t.over_6g = 1.0f / (6.0f * t.g);
  }
  return t;
}
// Eight codes of numbers times a factor.
__device__ __forceinline__ uint32_t e2m1_codes_times(const float* v, float f) {
  const float r[8] = {v[0] * f, v[1] * f, v[2] * f, v[3] * f, v[4] * f, v[5] * f, v[6] * f, v[7] * f};
  return e2m1_codes(r);
}
// Where a little less and a little more than a quotient round to different codes: the border between the two decides, by a comparison
// that is exact, since border * s has few bits and the fused product with g is rounded only after the subtraction.  (Numbers of few
// bits over a scale of few bits often lie on a border or next to it: with a tensor scale of 1 / 56, 16-bit numbers in one block
// of twelve.)  diff: the nibbles that differ; number(i): the lane's i-th number.
template <typename F>
__device__ __forceinline__ uint32_t settle_codes(uint32_t codes, uint32_t diff, float s, float g, float lift, F number) {
  while (diff) {
    const int at = (__ffs(static_cast<int>(diff)) - 1) & ~3;
    diff &= ~(15u << at);
    const uint32_t a = (codes >> at) & 7u;                     // the other one is a + 1
    const float border = 0.5f * (e2m1_magnitude(a) + e2m1_magnitude(a + 1u)) * s;
    const float r = fmaf(border, g, -fabsf(number(at >> 2)) * lift);
    if (r < 0.0f || (r == 0.0f && (a & 1u))) codes += 1u << at;
  }
  return codes;
}

// The block's scale byte and the codes of this lane's sixteen numbers: a block of block16, or half of one of block32, whose other half is
// the neighbouring lane's.  top: the largest magnitude of the lane's numbers, as bits (NaN is above infinity is above everything else).
// number(i): the lane's i-th number once more, for the few that need it.
template <int FORMAT, typename F>
__device__ __forceinline__ uint2 quantize_16(const float (&v)[16], uint32_t top, const TensorScale& t, uint32_t& byte, F number) {
  if (FORMAT == B2VX_FP4_BLOCK32) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const int e = static_cast<int>(top >> 23) - 2;            // biased exponent of 2^(floor(log2 amax) - 2)
    byte = static_cast<uint32_t>(max(e, 0));
    const float f = __uint_as_float((254u - min(byte, 253u)) << 23);   // a power of two: the products are exact
    uint2 codes = make_uint2(e2m1_codes_times(v, f), e2m1_codes_times(v + 8, f));
    if (top >= 0x7f800000u) {
      byte = 255u;
      codes = make_uint2(0u, 0u);
    }
    return codes;
  }
  // amax / (6 g) as a product of three roundings is off by less than 2^-22 of itself: where a little less and a little more round to
  // the same byte, that is the answer, else the border between them, as in settle_codes.
  constexpr float kLess = 1.0f - 0x1p-20f, kMore = 1.0f + 0x1p-20f;
  const float amax = __uint_as_float(top) * t.lift;
  const float q = amax * t.over_6g;
  const uint32_t two = e4m3_bytes(q * kLess, q * kMore);
  byte = two >> 8;
  if ((two & 0xff) != byte) {
    const float border6 = 3.0f * (e4m3_value(two & 0xff) + e4m3_value(byte));
    const float r = fmaf(border6, t.g, -amax);
    if (r > 0.0f || (r == 0.0f && (byte & 1u))) byte = two & 0xff;
  }
  const float s = e4m3_value(byte);
  float over_s;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(over_s) : "f"(s));   // off by 2^-23; s = 0 is dealt with below
  // The numbers over s g: the approximate reciprocal, two products and 1 / g are off by less than 2^-21 together.
  const float inv = over_s * t.over_g * t.lift, less = inv * kLess, more = inv * kMore;
  uint2 codes = make_uint2(e2m1_codes_times(v, less), e2m1_codes_times(v + 8, less));
  const uint2 up = make_uint2(e2m1_codes_times(v, more), e2m1_codes_times(v + 8, more));
  if ((codes.x != up.x || codes.y != up.y) && byte != 0) {
    codes.x = settle_codes(codes.x, codes.x ^ up.x, s, t.g, t.lift, number);
    codes.y = settle_codes(codes.y, codes.y ^ up.y, s, t.g, t.lift, [&](int i) { return number(8 + i); });
  }
  if (byte == 0) codes = make_uint2(0u, 0u);                  // every number rounds to zero
  if (top >= 0x7f800000u || !t.ok) {
    byte = 127u;
    codes = make_uint2(0u, 0u);
  }
  return codes;
}

}  // namespace b2vx
#endif  // B2VX_FP4_CUH_
