// Device code of the 4-bit cache format (fp4_cache.cu describes it): one
// group of 16 channels between 16-bit values and e2m1 values with a scale.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace fkv {

// x / d for 0 <= x < 2^28 and 0 < d <= 2^12 as one product: with 2^c >= d and
// mul = (2^(28 + c) + e) / d, 0 < e <= d, the product is x e / 2^(28 + c) of a
// d-th too large, less than one.  mul is at most 2^29.
struct Divisor {
  uint32_t mul;
  int shift;
};
inline Divisor divisor_of(int d) {
  int shift = 28;
  while (d > 1 << (shift - 28)) ++shift;
  return {(uint32_t)(((uint64_t)1 << shift) / d + 1), shift};
}
__device__ __forceinline__ int divide(int x, const Divisor &by) { return (int)(((uint64_t)(uint32_t)x * by.mul) >> by.shift); }

// The scale code nearest to v >= 0 (ties to the even code), at most 226,
// which is 10240: 6 * 10240 is below the largest half.
__device__ __forceinline__ uint32_t scale_code(float v) {
  uint32_t c;
  if (v < 6.103515625e-05f) {  // below 2^-14 the codes are multiples of 2^-17
    c = (uint32_t)__float2int_rn(v * 131072.0f);
  } else {
    uint32_t u = __float_as_uint(v);
    u += 0x7FFFFu + ((u >> 20) & 1);  // to 3 mantissa bits, ties to even
    c = (u >> 20) - ((127 - 15) << 3);
  }
  return c < 226 ? c : 226;
}

// amax / 6 for scale_code, exact where it decides: amax has at most 11
// significant bits, so the quotient either is a border of the scales (5 bits)
// or is 2^-11 of it away, and the product with 1/6, off by 2^-23, rounded to 15
// bits is on the same side, or the border itself.
__device__ __forceinline__ float sixth(float amax) {
  return __uint_as_float((__float_as_uint(amax * (1.0f / 6.0f)) + 0x100u) & ~0x1FFu);
}

// The half a scale code stands for, in both halves of a register.
__device__ __forceinline__ uint32_t scale_half2(uint32_t code) { return code * 0x00800080u; }

// The four bytes of a word, two e2m1 values each (low four bits first), as two halves.
__device__ __forceinline__ void e2m1x8_to_half2(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      " cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight floats to eight e2m1 values (a word, the first in the low bits):
// nearest, ties to even, saturating at 6.
__device__ __forceinline__ uint32_t floats_to_e2m1x8(const float (&y)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}

template <bool BF16>
__device__ __forceinline__ float2 pair_to_float2(uint32_t x) {
  if (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}

// Quantise 16 values (8 pairs); returns the scale code.
//
// x / s is formed as x * (1 / s) and passed through half precision, which
// makes the rounding to e2m1 exact: x has at most 11 significant bits and s
// 4, so x / s either is a tie between two e2m1 values or is at least 1/1920
// of it away.  The product is within 2^-22 of the quotient, so a tie becomes
// the tie itself in half (all seven ties are halves), and nothing else does
// (half a step of half precision is less than the distance: 1/2048 of the
// power of two below).
template <bool BF16>
__device__ __forceinline__ uint32_t quantise_group(uint32_t (&x)[8], uint2 &payload) {
  float amax;
  if (BF16) {
    __nv_bfloat162 m = __habs2(*reinterpret_cast<__nv_bfloat162 *>(&x[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<__nv_bfloat162 *>(&x[i])));
    amax = __bfloat162float(__hmax_nan(m.x, m.y));
  } else {
    __half2 m = __habs2(*reinterpret_cast<__half2 *>(&x[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<__half2 *>(&x[i])));
    amax = __half2float(__hmax_nan(m.x, m.y));
  }
  if (amax != amax) {  // NaN counts as zero: the format has none
    const uint32_t inf = BF16 ? 0x7F80u : 0x7C00u;
    amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if ((x[i] & 0x7FFFu) > inf) x[i] &= 0xFFFF0000u;
      if (((x[i] >> 16) & 0x7FFFu) > inf) x[i] &= 0x0000FFFFu;
      const float2 f = pair_to_float2<BF16>(x[i]);
      amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
  }
  const uint32_t code = scale_code(sixth(amax));
  if (code == 0) {  // amax / 6 rounds to nothing
    payload = make_uint2(0, 0);
    return 0;
  }
  const __half2 s2 = *reinterpret_cast<const __half2 *>(&(const uint32_t &)scale_half2(code));
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__low2float(s2)));
  uint32_t out[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pair_to_float2<BF16>(x[4 * j + i]);
      const float2 r = __half22float2(__floats2half2_rn(f.x * inv, f.y * inv));
      y[2 * i] = r.x, y[2 * i + 1] = r.y;
    }
    out[j] = floats_to_e2m1x8(y);
  }
  payload = make_uint2(out[0], out[1]);
  return code;
}

// 16 values (8 pairs) of a group; exact in either type.
template <bool BF16>
__device__ __forceinline__ void dequantise_group(uint2 payload, uint32_t code, uint32_t (&y)[8]) {
  const uint32_t s = scale_half2(code);
  uint32_t q[2][4];
  e2m1x8_to_half2(payload.x, q[0]);
  e2m1x8_to_half2(payload.y, q[1]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = hmul2(q[i / 4][i % 4], s);
    if (BF16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
      y[i] = *reinterpret_cast<const uint32_t *>(&b);
    } else {
      y[i] = h;
    }
  }
}

}  // namespace fkv
