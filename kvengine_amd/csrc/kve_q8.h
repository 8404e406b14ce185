// The 8-bit cache: its two code types and what a code stands for.
//
// A block of tokens of one kv head holds codes c and one scale s for K and one for V;
// a value is c s. Codes are int8 (-127 .. 127) or e4m3 (4 significant bits, at most
// 448, steps of 2^-9 below 2^-6).
#pragma once

#include "kve_common.h"

namespace kve {

enum class Q8 { kInt8, kE4m3 };

constexpr float kInt8Max = 127.0f, kE4m3Max = 448.0f;
// The least scale of a block that is not all zeros: far above the smallest 32-bit
// numbers, so that quotients, reciprocals and products with codes stay normal.
constexpr float kMinScale = 0x1p-100f;

// The scale of a block whose largest finite value is amax. int8: amax / 127. e4m3: the
// least power of two that brings amax to 448 = 0.875 * 2^9 or below, for a code with an
// exponent gains nothing from a finer scale, and with powers of two a scale that grows
// later changes no code but the smallest (steps below 2^-6).
template <Q8 Q>
__device__ __forceinline__ float q8_scale(float amax) {
  if (!(amax > 0.0f)) return 0.0f;
  if constexpr (Q == Q8::kInt8) {
    return fmaxf(amax / kInt8Max, kMinScale);
  } else {
    int e;
    const float m = frexpf(amax, &e);
    return ldexpf(1.0f, max(e - 9 + (m > 0.875f ? 1 : 0), -100));
  }
}

// The reciprocal that q8_code takes.
__device__ __forceinline__ float q8_inv(float s) { return s > 0.0f ? 1.0f / s : 0.0f; }

// x / s to the nearest int8, ties to even, of the exact quotient: the product with the
// reciprocal may be off by 2^-23 of it, so the two borders beside the rounded number are
// tested by one fma each, whose sign is exact.
__device__ __forceinline__ float int8_code(float x, float s, float inv) {
  float n = rintf(x * inv);
  n = fminf(fmaxf(n, -kInt8Max), kInt8Max);
  const float up = fmaf(-(n + 0.5f), s, x), dn = fmaf(-(n - 0.5f), s, x);
  const bool odd = static_cast<int>(n) & 1;
  if (up > 0.0f || (up == 0.0f && odd)) n += 1.0f;
  else if (dn < 0.0f || (dn == 0.0f && odd)) n -= 1.0f;
  return fminf(fmaxf(n, -kInt8Max), kInt8Max);
}

// Codes of four values against a scale (inv of it), the first in the lowest byte. NaN
// becomes 0 and an infinity the largest code (0 where the scale is 0).
template <Q8 Q>
__device__ __forceinline__ uint32_t q8_codes(const float (&x)[4], float s, float inv) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] == x[i] && inv > 0.0f ? x[i] : 0.0f;
  if constexpr (Q == Q8::kInt8) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r |= (static_cast<uint32_t>(static_cast<int>(int8_code(y[i], s, inv))) & 0xffu) << (8 * i);
    return r;
  } else {
    // (a power of two's reciprocal is exact)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(y[i] * inv, -kE4m3Max), kE4m3Max);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true));
  }
}

// What byte i of a word stands for before its scale.
template <Q8 Q, int I>
__device__ __forceinline__ float q8_value(uint32_t w) {
  if constexpr (Q == Q8::kInt8)
    return static_cast<float>(static_cast<int8_t>(w >> (8 * I)));
  else
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), I);
}

// Four codes of a block whose scale goes from s0 to s, to the nearest, ties to even. In
// 64 bits: c s0 has up to 32, and no quotient of two such lies nearer a border than 2^-33
// without being on it.
template <Q8 Q>
__device__ __forceinline__ uint32_t q8_rescale(uint32_t w, float s0, float s) {
  const double f[4] = {q8_value<Q, 0>(w), q8_value<Q, 1>(w), q8_value<Q, 2>(w), q8_value<Q, 3>(w)};
  uint32_t r = 0;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double v = s > 0.0f ? f[i] * s0 / s : 0.0;
    if constexpr (Q == Q8::kInt8)
      r |= (static_cast<uint32_t>(static_cast<int>(fmin(fmax(rint(v), -127.0), 127.0))) & 0xffu)
           << (8 * i);
    else
      y[i] = static_cast<float>(v == v ? fmin(fmax(v, -448.0), 448.0) : v);  // (a NaN stays)
  }
  if constexpr (Q == Q8::kInt8) {
    return r;
  } else {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true));
  }
}

}  // namespace kve
