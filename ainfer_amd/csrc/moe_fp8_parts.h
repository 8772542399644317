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
//
// The fp32 quotient is the correctly rounded one, without a division for each value: from r,
// the rounded 1 / s, v r is within two units of the last place, and each step q + (v - q s) r
// brings it nearer until the second one rounds correctly (P. Markstein, Computation of
// elementary functions on the IBM RISC System/6000 processor, 1990).  The remainders are exact
// while no bit of theirs is under fp32's 2^-149: quotients that decide on a code are 2^-11 or
// more, so their last bits times s's are 2^-34-23 s or more.  Below s = 2^-90 the values are
// divided.  An infinite s takes r = 0 and no remainder: finite values become 0.
template <int N>
__device__ __forceinline__ void fp8_codes(const float (&v)[N], float s, uint32_t (&q)[N / 4]) {
  float x[N];
  if (s < 0x1p-90f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i] / s;
  } else {
    const float r = 1.0f / s, d = s == INFINITY ? 0.0f : s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float y = v[i] * r;
      y = fmaf(fmaf(-y, d, v[i]), r, y);
      x[i] = copysignf(fmaf(fmaf(-y, d, v[i]), r, y), v[i]);  // -0 stays -0
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
    q[i] = (uint32_t)w;
  }
}

// g / (1 + exp(-g)) * u to 2^-21 of itself and 2^-119 of u: exp(-g) as 2^(h + l), h + l = -g
// log2 e with the rounding of h in l, by the hardware's exp2 and a factor 1 + l ln 2 (3 2^-24
// together), the sum 2^-24, the hardware's reciprocal 2^-23 and two products 2^-24 each.  The
// exponent's g is kept within +-200, where exp(-g) is 0 or infinite; from exp(-g) = 2^126 on the
// reciprocal may be 0 (g 2^-126 is what is lost, g being -87 to -89 there, and less below).
// (With silu_mul's expf and division, and a division for each code, 32768 x 1024 bf16 took 56.8
// us, now 40.4.)
__device__ __forceinline__ float silu_mul_near(float g, float u) {
  const float c = fminf(fmaxf(g, -200.0f), 200.0f);
  const float h = c * -1.44269502162933349609f;             // -log2 e, rounded
  const float l = fmaf(c, -1.44269502162933349609f, -h) + c * -1.92596299112661746e-8f;
  float e = __builtin_amdgcn_exp2f(h);
  e = fminf(fmaf(e, l * 0.69314718056f, e), INFINITY);  // an infinite e stays one (no NaN)
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

}  // namespace
