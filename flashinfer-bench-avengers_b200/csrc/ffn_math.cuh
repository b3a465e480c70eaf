// Element arithmetic of the dense feed-forward block and of 4-bit
// microscaled blocks, shared by its kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace moe {

// Activation codes and 16/32-bit type codes (moe_b200.h).
constexpr int kActSilu = 0;
constexpr int kActGeluTanh = 1;
constexpr int kTypeBf16 = 0;
constexpr int kTypeFp16 = 1;
constexpr int kTypeFp32 = 2;

// Both activations are g * s with s = 1 / (1 + exp(-q(g))): q = g for SiLU,
// and q = 2 c (g + 0.044715 g^3), c = sqrt(2 / pi), for the tanh form of
// GELU, because (1 + tanh z) / 2 is the logistic function of 2 z (this form
// does not cancel where tanh is near -1). The fast exponential is off by up to
// 2 + 1.173 |q| units in the last place, the division by 2, and rounding q
// itself adds up to 2 |q| in the tanh form: s is good to (5 + 3.2 |q|) 2^-23 of
// its value for negative q (5e-6 at q = -10, 3e-5 at -80, where s is 2e-35), and
// to a few 2^-23 for positive q, where the exponential is small beside the 1.
// Against g that is at most 3e-7, far below the 16-bit results' 2^-9.
__device__ __forceinline__ float act_gate(float g, int act) {
  const float q = act == kActSilu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return __fdividef(1.0f, 1.0f + __expf(-q));
}

__device__ __forceinline__ float act_value(float g, int act) { return g * act_gate(g, act); }

// act(g) and its derivative s + g s (1 - s) q'(g). Where s (1 - s) has
// rounded to zero the second term is zero, also where g or q' is infinite.
__device__ __forceinline__ void act_value_slope(float g, int act, float& value, float& slope) {
  const float s = act_gate(g, act);
  const float dq = act == kActSilu ? 1.0f : 1.5957691216057308f * (1.0f + 0.134145f * g * g);
  const float curve = s * (1.0f - s);
  value = g * s;
  slope = curve == 0.0f ? s : s + g * curve * dq;
}

__device__ __forceinline__ uint32_t pack_16(float lo, float hi, int type) {
  if (type == kTypeBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float2 unpack_16(uint32_t bits, int type) {
  if (type == kTypeBf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&bits));
  return __half22float2(*reinterpret_cast<const __half2*>(&bits));
}

// A value in two 16-bit parts is v rounded, and what that left times
// rest_scale, rounded again; the reader's fp32 sums of the second part are
// multiplied by rest_unscale. fp16 needs the factor: its smallest step is 2^-24,
// so that less than 11 bits are left of the rest of a value below 2^-3 and
// nothing below 2^-14 (error of dx at 16 tokens, H = 1024, I = 512, output
// gradients of 1e-4, 1e-5 and 1e-6: 2.9e-4 -> 2.1e-4, 2.0e-3 -> 2.2e-4 and
// 2.0e-2 -> 1.3e-3, what rounding dx to fp16 alone gives; same time).
// A rest is at most 16, half a step at fp16's largest, so that 2^11 of it fit.
// bf16 has fp32's range.
__device__ __forceinline__ float rest_scale(int type) { return type == kTypeFp16 ? 2048.0f : 1.0f; }
__device__ __forceinline__ float rest_unscale(int type) { return type == kTypeFp16 ? 1.0f / 2048.0f : 1.0f; }

// The second parts of (lo, hi), whose first are `packed`: 0 beside an infinity,
// so that a value beyond the type stays infinite in a sum of both.
__device__ __forceinline__ uint32_t pack_rest_16(float lo, float hi, uint32_t packed, int type) {
  const float2 v = unpack_16(packed, type);
  const float f = rest_scale(type);
  return pack_16(isinf(v.x) ? 0.f : (lo - v.x) * f, isinf(v.y) ? 0.f : (hi - v.y) * f, type);
}

// ------------------------------------------------- 4-bit microscaled blocks
// Exponent byte of a block from the largest magnitude's bits: floor(log2) - 2
// (the largest e2m1 exponent), biased by 127, at least 0. Infinities and
// NaNs give 255, the NaN exponent, and 255 stays the only byte above 252.
__device__ __forceinline__ uint32_t mx_exponent(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// 2^(127 - byte): the factor that brings a block into e2m1's range. A power
// of two, so the product is exact wherever it matters for rounding.
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Eight values times `inv`, rounded to e2m1 (nearest, ties to even, beyond 6
// to 6), the first in the lowest nibble.
__device__ __forceinline__ uint32_t mx_pack8(const float* v, float inv) {
  uint32_t r;
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n\t"
      "mov.b32 %0, {t0, t1, t2, t3};\n\t}"
      : "=r"(r)
      : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
        "f"(v[6] * inv), "f"(v[7] * inv));
  return r;
}

// Byte of row r, 32-column block b in the tiled exponent array of a matrix
// with `k_tiles` = ceil(K / 128) tiles per 128 rows.
__host__ __device__ __forceinline__ int64_t mx_scale_offset(int64_t r, int64_t b, int64_t k_tiles) {
  return ((r >> 7) * k_tiles + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

}  // namespace moe
