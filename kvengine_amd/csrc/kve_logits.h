// Reading rows of logits for the kernels that go over whole vocabularies: a wave's
// chunk as 16-byte vectors at any alignment, and reductions that keep a NaN.
#pragma once

#include "kve_common.h"

#include <type_traits>

namespace kve {

constexpr int kChunk = 2048;  // logits: 32 per lane of a wave, 8 per thread of 256

// (v_maximum / v_minimum: a NaN stays, so that it reaches the sums)
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// over the 16 lanes of a row
__device__ __forceinline__ float row_max(float v) {
  v = max_nan(v, dpp_mov<0xB1>(v));
  v = max_nan(v, dpp_mov<0x4E>(v));
  v = max_nan(v, dpp_mov<0x141>(v));
  return max_nan(v, dpp_mov<0x140>(v));
}
__device__ __forceinline__ double row_sum(double v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  v = row_max(v);
  const uint32_t u = __float_as_uint(v);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = max_nan(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const uint32_t w = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return max_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v = row_sum(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

template <typename E>
__device__ __forceinline__ float to_f32(E v) {
  if constexpr (std::is_same_v<E, float>) return v;
  else return bf16_to_f32(v);
}

template <typename E>
constexpr int kVec = 16 / sizeof(E);

// A 16-byte vector of logits as stored, from element i0 on, of a row of V; those past the
// end are -inf. Rows may start at any element (an odd vocabulary): gfx950 reads vectors
// at the type's alignment.
template <typename E>
__device__ __forceinline__ u32x4 load_raw(const E* row, int i0, int V) {
  constexpr int N = kVec<E>;
  struct __attribute__((packed, aligned(sizeof(E)))) Vec { u32x4 v; };
  if (i0 + N <= V) return reinterpret_cast<const Vec*>(row + i0)->v;
  u32x4 x;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (N == 4) {
      x[w] = i0 + w < V ? __float_as_uint(row[i0 + w]) : 0xff800000u;
    } else {
      const uint32_t lo = i0 + 2 * w < V ? row[i0 + 2 * w] : 0xff80u;
      const uint32_t hi = i0 + 2 * w + 1 < V ? row[i0 + 2 * w + 1] : 0xff80u;
      x[w] = lo | hi << 16;
    }
  }
  return x;
}

// Logit e of such a vector.
template <typename E>
__device__ __forceinline__ float logit(const u32x4& x, int e) {
  if constexpr (kVec<E> == 4) return __uint_as_float(x[e]);
  else return __uint_as_float(e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
}

template <typename E>
__device__ __forceinline__ void load_logits(const E* row, int i0, int V, float (&x)[kVec<E>]) {
  const u32x4 raw = load_raw<E>(row, i0, V);
#pragma unroll
  for (int e = 0; e < kVec<E>; ++e) x[e] = logit<E>(raw, e);
}

// A lane's share of a chunk as stored: logits ch * kChunk + v * 64 * N + lane * N ...
template <typename E>
struct Piece {
  static constexpr int N = kVec<E>, NV = kChunk / (64 * N);
  u32x4 x[NV];
  __device__ __forceinline__ void load(const E* row, int ch, int l, int V) {
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v] = load_raw<E>(row, (ch * NV + v) * 64 * N + l * N, V);
  }
  // Vector v from here on only: without it the compiler converts every logit of the
  // chunk ahead of the sums (120 registers, four waves a SIMD).
  __device__ __forceinline__ void hide(int v) { __asm__ volatile("" : "+v"(x[v])); }
};

}  // namespace kve
