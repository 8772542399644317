// moe_fp8_parts.h - device pieces of the 8-bit floating point operators
// (moe_fp8.hip, moe_fp8_product.hip, moe_sort.hip): rows at any alignment of
// their elements, the scale of a group and its e4m3 codes.
#pragma once
#include "moe_common.h"

namespace {

// vectors at any address of their elements: rows of an odd length or pitch are read
// in 16-byte pieces as well (the hardware's unaligned global accesses)
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

// N consecutive values of a row (N a multiple of 8)
template <bool F32, int N>
__device__ __forceinline__ void load_row(const void *p, int64_t at, float (&v)[N]) {
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 a = *(const f32x4_any *)((const float *)p + at + i);
#pragma unroll
      for (int d = 0; d < 4; ++d) v[i + d] = a[d];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const u32x4 a = *(const u32x4_any *)((const uint16_t *)p + at + i);
#pragma unroll
      for (int d = 0; d < 8; ++d)
        v[i + d] = __uint_as_float(d & 1 ? a[d / 2] & 0xFFFF0000u : a[d / 2] << 16);
    }
  }
}
template <bool F32>
__device__ __forceinline__ float load_one(const void *p, int64_t at) {
  return F32 ? ((const float *)p)[at] : bf16_to_f32(((const uint16_t *)p)[at]);
}
template <bool F32, int N, bool NT = false>
__device__ __forceinline__ void store_row(void *p, int64_t at, const float (&v)[N]) {
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 w = {v[i], v[i + 1], v[i + 2], v[i + 3]};
      if constexpr (NT) __builtin_nontemporal_store(w, (f32x4_any *)((float *)p + at + i));
      else *(f32x4_any *)((float *)p + at + i) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      u32x4 w;
#pragma unroll
      for (int d = 0; d < 4; ++d) w[d] = bf16x2_bits(v[i + 2 * d], v[i + 2 * d + 1]);
      if constexpr (NT) __builtin_nontemporal_store(w, (u32x4_any *)((uint16_t *)p + at + i));
      else *(u32x4_any *)((uint16_t *)p + at + i) = w;
    }
  }
}
template <bool F32>
__device__ __forceinline__ void store_one(void *p, int64_t at, float v) {
  if constexpr (F32) ((float *)p)[at] = v;
  else ((uint16_t *)p)[at] = f32_to_bf16(v);
}

// The scale of a group whose largest magnitude is m: m / 448 (448 is e4m3's largest
// value), at least the smallest normal fp32 value, 1 for a group of zeros; pow2:
// the least power of two that is not below it.  An infinite m gives an infinite scale.
__device__ __forceinline__ float fp8_scale(float m, bool pow2) {
  if (m == 0.0f) return 1.0f;
  float s = fmaxf(m / 448.0f, 0x1p-126f);
  if (pow2) {
    uint32_t u = __float_as_uint(s);
    if (u & 0x007FFFFFu) u = (u & 0x7F800000u) + 0x00800000u;
    s = __uint_as_float(u);
  }
  return s;
}
// the larger one; a NaN b leaves a
__device__ __forceinline__ float max_skip_nan(float a, float b) { return b > a ? b : a; }
// the largest of 8 neighbouring lanes' m >= 0, in all of them
__device__ __forceinline__ float max_of_8_lanes(float m) {
  auto step = [&](auto ctrl) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(
        0, (int)__float_as_uint(m), decltype(ctrl)::value, 0xF, 0xF, false);
    m = fmaxf(m, __uint_as_float(o));
  };
  step(std::integral_constant<int, 0xB1>());   // lanes ^ 1
  step(std::integral_constant<int, 0x4E>());   // lanes ^ 2
  step(std::integral_constant<int, 0x141>());  // the other four of the eight
  return m;
}
// e4m3 codes of v / s, nearest even.  |v / s| is at most 448 (1 + 2^-23) by the scale's
// choice, so no conversion overflows; NaN (and inf / inf) become e4m3's NaN.
template <int N>
__device__ __forceinline__ void fp8_codes(const float (&v)[N], float s, uint32_t (&q)[N / 4]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] / s, v[4 * i + 1] / s, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] / s, v[4 * i + 3] / s, w, true);
    q[i] = (uint32_t)w;
  }
}

}  // namespace
