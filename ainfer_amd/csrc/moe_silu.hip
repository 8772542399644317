// moe_silu.hip - the gated activation between an MLP's projections
// (ainfer_moe_silu_mul): act = g / (1 + exp(-g)) * u, rows of any pitch.
// One pass, bound by memory: two inputs read, one output written.
#include "moe_common.h"
#include "moe_internal.h"

namespace {

// 8 elements from p: 16 (bf16) or 2 x 16 (fp32) bytes, or one by one
template <bool F32, bool VEC>
__device__ __forceinline__ void load8(const void *p, int64_t at, int n, float (&v)[8]) {
  if constexpr (VEC && F32) {
    const f32x4 a = *(const f32x4 *)((const float *)p + at);
    const f32x4 b = *(const f32x4 *)((const float *)p + at + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else if constexpr (VEC) {
    const u32x4 a = *(const u32x4 *)((const uint16_t *)p + at);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = __uint_as_float(i & 1 ? a[i / 2] & 0xFFFF0000u : a[i / 2] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n)
        v[i] = F32 ? ((const float *)p)[at + i] : bf16_to_f32(((const uint16_t *)p)[at + i]);
      else
        v[i] = 0.0f;
  }
}

// VEC: every row and its length allow 16-byte accesses
template <bool IF32, bool OF32, bool VEC>
__global__ __launch_bounds__(256) void k_silu_rows(const void *g, int64_t gld, const void *u,
                                                   int64_t uld, void *y, int64_t yld, int64_t n8,
                                                   int64_t per_row, int64_t I) {
  for (int64_t c = blockIdx.x * 256ll + threadIdx.x; c < n8; c += gridDim.x * 256ll) {
    const int64_t row = per_row == n8 ? 0 : c / per_row;
    const int64_t col = (c - row * per_row) * 8;
    const int n = (int)(I - col < 8 ? I - col : 8);
    float gv[8], uv[8];
    load8<IF32, VEC>(g, row * gld + col, n, gv);
    load8<IF32, VEC>(u, row * uld + col, n, uv);
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = silu_mul(gv[i], uv[i]);
    const int64_t at = row * yld + col;
    if constexpr (VEC && OF32) {
      float *p = (float *)y + at;
      *(f32x4 *)p = (f32x4){o[0], o[1], o[2], o[3]};
      *(f32x4 *)(p + 4) = (f32x4){o[4], o[5], o[6], o[7]};
    } else if constexpr (VEC) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)f32_to_bf16(o[2 * i]) | ((uint32_t)f32_to_bf16(o[2 * i + 1]) << 16);
      *(u32x4 *)((uint16_t *)y + at) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) {
          if (OF32)
            ((float *)y)[at + i] = o[i];
          else
            ((uint16_t *)y)[at + i] = f32_to_bf16(o[i]);
        }
    }
  }
}

}  // namespace

hipError_t launch_silu_rows(const void *g, int64_t gld, const void *u, int64_t uld, int in_dtype,
                            int T, int I, void *y, int64_t yld, int out_dtype, hipStream_t s) {
  const bool i32 = in_dtype == AINFER_ACT_F32, o32 = out_dtype == AINFER_ACT_F32;
  const int isz = i32 ? 4 : 2, osz = o32 ? 4 : 2;
  int64_t rows = T, cols = I;
  if (gld == I && uld == I && yld == I) {  // one long row
    cols *= rows;
    rows = 1;
  }
  auto al = [&](const void *p, int64_t ld, int sz) {
    return (uintptr_t)p % 16 == 0 && (rows == 1 || (ld * sz) % 16 == 0);
  };
  const bool vec = cols % 8 == 0 && al(g, gld, isz) && al(u, uld, isz) && al(y, yld, osz);
  const int64_t per = (cols + 7) / 8, n8 = per * rows;
  const int64_t blocks = (n8 + 255) / 256;
  const int grid = (int)(blocks < 4096 ? blocks : 4096);
#define SILU(A, B, V) \
  k_silu_rows<A, B, V><<<grid, 256, 0, s>>>(g, gld, u, uld, y, yld, n8, per, cols)
  if (i32 && o32) { if (vec) SILU(true, true, true); else SILU(true, true, false); }
  else if (i32) { if (vec) SILU(true, false, true); else SILU(true, false, false); }
  else if (o32) { if (vec) SILU(false, true, true); else SILU(false, true, false); }
  else { if (vec) SILU(false, false, true); else SILU(false, false, false); }
#undef SILU
  return hipGetLastError();
}
