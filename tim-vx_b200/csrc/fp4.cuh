// Conversions of 4-bit block floating point: e2m1 codes, e8m0 and e4m3 scales.
#ifndef B2VX_FP4_CUH_
#define B2VX_FP4_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "b2vx.h"

namespace b2vx {

// Eight floats to e2m1 codes (nearest even, cut to +-6), element i in bits 4 i.
__device__ __forceinline__ uint32_t e2m1_codes(const float* v) {
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

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Sixteen numbers from column c on, zeros from column k on, as they lie.  VEC: rows start on 16 bytes, so whole pieces load in 16 bytes.
template <typename T>
struct alignas(16) Sixteen {
  T v[16];
};
template <typename T, bool VEC>
__device__ __forceinline__ Sixteen<T> load_16(const T* row, int c, int k, uint4* staging, int lane) {
  Sixteen<T> t;
  constexpr int W = sizeof(t) / 16;
  if (VEC && c + 16 <= k) {
    const uint4* src = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(&t)[i] = __ldg(src + i);
  } else if (VEC) {
#pragma unroll
    for (int i = 0; i < 16; ++i) t.v[i] = c + i < k ? row[c + i] : from_float<T>(0.0f);
  } else {
    // neighbouring numbers by neighbouring lanes, handed over through the warp's staging memory: each lane's sixteen numbers and 16 bytes
    // more, so that eight lanes' 16-byte pieces fall into different banks
    constexpr int kPitch = 16 + 16 / sizeof(T);
    T* s = reinterpret_cast<T*>(staging);
    const int first = c - lane * 16;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int at = i * 32 + lane;
      s[(at >> 4) * kPitch + (at & 15)] = first + at < k ? row[first + at] : from_float<T>(0.0f);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(&t)[i] = staging[lane * (W + 1) + i];
  }
  return t;
}
template <typename T>
__device__ __forceinline__ Sixteen<T> load_whole(const T* from) {
  Sixteen<T> t;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(t) / 16); ++i) reinterpret_cast<uint4*>(&t)[i] = __ldg(reinterpret_cast<const uint4*>(from) + i);
  return t;
}
// The largest magnitude, as float bits.
template <typename T>
__device__ __forceinline__ uint32_t top_of(const Sixteen<T>& t) {
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(t.v[i]) & 0x7fffffffu);
    return top;
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&t);
    constexpr uint32_t kMagnitudes = 0x7fff7fffu;
    uint32_t two = w[0] & kMagnitudes;
#pragma unroll
    for (int i = 1; i < 7; i += 2) two = __vimax3_u16x2(two, w[i] & kMagnitudes, w[i + 1] & kMagnitudes);
    two = __vmaxu2(two, w[7] & kMagnitudes);
    const uint32_t top = max(two & 0xffffu, two >> 16);
    if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top)))) & 0x7fffffffu;
    else return top << 16;
  }
}

// What quantization needs of block16's tensor scale, worked out once by a thread.
struct TensorScale {
  float g = 1.0f;          // times lift
  float lift = 1.0f;       // numbers are multiplied by it: near the ends of float's range nothing then overflows or loses bits
  float over_g = 1.0f;     // 1 / g
  float over_6g = 1.0f;    // 1 / (6 g)
  bool ok = true;
  uint32_t near = 3;       // below
};
// Numbers over s g are rounded to codes from an approximate quotient, which can only go wrong next to a border between two codes.  For
// 16-bit numbers the places where that can happen are few and known beforehand: a number lies within 2^-19 of a border b s g only
// if b s g itself is that close to a number of the 16-bit type, which depends on the mantissas of b (1, 1.25, 1.5 or 1.75), s (eight
// of them) and g alone.  Lane i works out, for the i-th mantissa of s, whether such numbers lie below their border (bit 0: a
// quotient that is a little too small is right), above it (bit 1: one a little too large) or on it (both bits).
template <typename T>
__device__ __forceinline__ uint32_t near_borders(float g) {
  if (sizeof(T) == 4) return 3u;
  const float gn = __uint_as_float((__float_as_uint(g) & 0x7fffffu) | 0x3f800000u);
  uint32_t near = 0;
#pragma unroll
  for (int m = 4; m < 8; ++m) {
    const float p = 0.25f * m * (1.0f + 0.125f * (threadIdx.x & 7));      // few bits: exact
    float v;
    if constexpr (std::is_same<T, __half>::value) v = __half2float(__float2half_rn(p * gn));
    else v = __bfloat162float(__float2bfloat16_rn(p * gn));
    const float r = fmaf(p, gn, -v);                                      // its sign is exact
    if (fabsf(r) <= 0x1p-19f * v) near |= r > 0.0f ? 1u : (r < 0.0f ? 2u : 3u);
  }
  return near;
}
template <int FORMAT, typename T>
__device__ __forceinline__ TensorScale tensor_scale(const float* p) {
  TensorScale t;
  if (FORMAT == B2VX_FP4_BLOCK16) {
    const float g = __ldg(p);
    t.ok = g > 0.0f && g < __int_as_float(0x7f800000);
    t.lift = g < 0x1p-60f ? 0x1p64f : (g > 0x1p60f ? 0x1p-64f : 1.0f);
    t.g = g * t.lift;
    t.over_g = 1.0f / t.g;
    t.over_6g = 1.0f / (6.0f * t.g);
    t.near = near_borders<T>(t.g);
  }
  return t;
}
// Eight codes of numbers times a factor.
__device__ __forceinline__ uint32_t e2m1_codes_times(const float* v, float f) {
  const float r[8] = {v[0] * f, v[1] * f, v[2] * f, v[3] * f, v[4] * f, v[5] * f, v[6] * f, v[7] * f};
  return e2m1_codes(r);
}
// Where a little less and a little more than a quotient round to different codes: the border between the two decides, by a comparison
// that is exact, since border * s has few bits and the fused product with g is rounded only after the subtraction.  diff: the nibbles that differ; number(i): the lane's i-th number.
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
// the neighbouring lane's.  number(i): the lane's i-th number once more, for the few that need it.
template <int FORMAT, typename T, typename F>
__device__ __forceinline__ uint2 quantize_16(const Sixteen<T>& x, const TensorScale& t, uint32_t& byte, F number) {
  uint32_t top = top_of(x);         // as bits: NaN is above infinity is above everything else
  float v[16];
  if constexpr (FORMAT == B2VX_FP4_BLOCK32) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const int e = static_cast<int>(top >> 23) - 2;            // biased exponent of 2^(floor(log2 amax) - 2)
    byte = static_cast<uint32_t>(max(e, 0));
    const float f = __uint_as_float((254u - min(byte, 253u)) << 23);   // a power of two: the products are exact
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = to_float(x.v[i]) * f;
    uint2 codes = make_uint2(e2m1_codes(v), e2m1_codes(v + 8));
    if (top >= 0x7f800000u) {
      byte = 255u;
      codes = make_uint2(0u, 0u);
    }
    return codes;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = to_float(x.v[i]);
    if (t.lift != 1.0f) {             // else the factor below could overflow: s g may be less than 2^-128
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= t.lift;
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
    const float inv = over_s * t.over_g, less = inv * kLess, more = inv * kMore;
    const uint32_t near = __shfl_sync(0xffffffffu, t.near, (__float_as_uint(s) >> 20) & 7);
    const float f = near == 2u ? more : less;
    uint2 codes = make_uint2(e2m1_codes_times(v, f), e2m1_codes_times(v + 8, f));
    if (near == 3u) {
      const uint2 up = make_uint2(e2m1_codes_times(v, more), e2m1_codes_times(v + 8, more));
      if ((codes.x != up.x || codes.y != up.y) && byte != 0) {
        codes.x = settle_codes(codes.x, codes.x ^ up.x, s, t.g, t.lift, number);
        codes.y = settle_codes(codes.y, codes.y ^ up.y, s, t.g, t.lift, [&](int i) { return number(8 + i); });
      }
    }
    if (byte == 0) codes = make_uint2(0u, 0u);                  // every number rounds to zero
    if (top >= 0x7f800000u || !t.ok) {
      byte = 127u;
      codes = make_uint2(0u, 0u);
    }
    return codes;
  }
}

// Four neighbouring blocks' bytes as a word, in the first of their lanes.
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_word(uint32_t byte) {
  constexpr int LANES = FORMAT == B2VX_FP4_BLOCK32 ? 2 : 1;
  uint32_t word = byte | __shfl_down_sync(0xffffffffu, byte, LANES) << 8;
  word |= __shfl_down_sync(0xffffffffu, word, 2 * LANES) << 16;
  return word;
}

}  // namespace b2vx
#endif  // B2VX_FP4_CUH_
