// moe_fp8.hip - rows and weights quantised to e4m3 with a scale for each block of
// 128 (ainfer_moe_act_quant_fp8, ainfer_moe_weight_quant_fp8), and the gated
// activation written so (ainfer_moe_silu_mul_fp8): s = max |x| / 448, q = e4m3(x / s).
//
// One pass, bound by memory (a large copy reaches 4.95 TB/s): a group's values stay in its
// lanes' registers between the maximum and the codes.  32768 x 4096 bf16 79 us, 5.1 TB/s; fp32
// 129, 5.2; the gated activation of 32768 x 1024 bf16 40, 4.2 (the
// activation's instructions come on top), fp32 56, 5.4; 64 x 2048 x 4096 bf16 weights 300,
// 5.4.  128 x 512: 3.5 us, an empty launch takes 2.5.
// The codes are written through the caches: past them 32768 x 1024 takes 35 us, but with the
// product that reads the codes 236 instead of 220.
#include "moe_common.h"
#include "moe_internal.h"
#include "moe_fp8_parts.h"

namespace {

// 8 neighbouring lanes take the 128 columns of a group, 16 each (K is a multiple of
// 16, so a lane's columns are all inside the row or all behind it).
// SILU: the values are silu(x) * up.
template <bool F32, bool SILU>
__global__ __launch_bounds__(256) void k_quant_rows(const void *x, int64_t xld, const void *up,
                                                    int64_t uld, const int32_t *live, int N, int K,
                                                    int pow2, uint8_t *q, int64_t qld, float *sq) {
  const int G = (K + 127) / 128;
  const int rows = live ? max(0, min(*live, N)) : N;
  const int64_t items = (int64_t)rows * G * 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t row = i / (G * 8);
    const int col = (int)(i - row * (G * 8)) * 16;
    float v[16];
    if (col < K) {
      load_row<F32>(x, row * xld + col, v);
      if constexpr (SILU) {
        float u[16];
        load_row<F32>(up, row * uld + col, u);
#pragma unroll
        for (int d = 0; d < 16; ++d) v[d] = silu_mul_near(v[d], u[d]);
      }
    } else {
#pragma unroll
      for (int d = 0; d < 16; ++d) v[d] = 0.0f;
    }
    float m = 0.0f;
#pragma unroll
    for (int d = 0; d < 16; ++d) m = max_skip_nan(m, fabsf(v[d]));
    const float s = fp8_scale(max_of_8_lanes(m), pow2);
    if (col < K) {
      uint32_t w[4];
      fp8_codes(v, s, w);
      *(u32x4 *)(q + row * qld + col) = u32x4{w[0], w[1], w[2], w[3]};
    }
    if ((threadIdx.x & 7) == 0) sq[row * G + col / 128] = s;
  }
}

// One workgroup takes a block of 128 x 128 weights: lane c of 8 takes 16 columns of
// four rows, 32 apart.
template <bool F32>
__global__ __launch_bounds__(256) void k_quant_weights(const void *w, int M, int K, int pow2,
                                                       uint8_t *q, float *scales) {
  __shared__ float part[4];
  const int G = (K + 127) / 128, MB = (M + 127) / 128;
  const int64_t b = blockIdx.x;
  const int64_t e = b / ((int64_t)MB * G);
  const int rb = (int)(b / G % MB), cb = (int)(b % G);
  const int r0 = rb * 128 + threadIdx.x / 8, col = cb * 128 + (threadIdx.x & 7) * 16;
  float v[4][16], m = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 32 * i;
    if (r < M && col < K) {
      load_row<F32>(w, (e * M + r) * K + col, v[i]);
    } else {
#pragma unroll
      for (int d = 0; d < 16; ++d) v[i][d] = 0.0f;
    }
#pragma unroll
    for (int d = 0; d < 16; ++d) m = max_skip_nan(m, fabsf(v[i][d]));
  }
  m = __uint_as_float(wave_max_u32(__float_as_uint(m)));  // m >= 0: its bits are ordered
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  const float s = fp8_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), pow2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 32 * i;
    if (r < M && col < K) {
      uint32_t c[4];
      fp8_codes(v[i], s, c);
      *(u32x4 *)(q + (e * M + r) * K + col) = u32x4{c[0], c[1], c[2], c[3]};
    }
  }
  if (threadIdx.x == 0) scales[b] = s;
}

template <bool SILU>
hipError_t quant_rows(const void *x, int64_t xld, const void *up, int64_t uld, int dtype,
                      const int32_t *live, int N, int K, int scale_kind, uint8_t *q, int64_t qld,
                      float *sq, hipStream_t s) {
  const int64_t items = (int64_t)N * ((K + 127) / 128) * 8, blocks = (items + 255) / 256;
  const int grid = (int)(blocks < 4096 ? blocks : 4096);
  const int pow2 = scale_kind == AINFER_FP8_SCALE_POW2;
  return enqueue(dtype == AINFER_ACT_F32 ? k_quant_rows<true, SILU> : k_quant_rows<false, SILU>, grid,
                 256, s, x, xld, up, uld, live, N, K, pow2, q, qld, sq);
}

}  // namespace

hipError_t launch_act_quant_fp8(const void *x, int64_t xld, int dtype, const int32_t *live, int N,
                                int K, int scale_kind, uint8_t *q, int64_t qld, float *sq,
                                hipStream_t s) {
  return quant_rows<false>(x, xld, nullptr, 0, dtype, live, N, K, scale_kind, q, qld, sq, s);
}

hipError_t launch_silu_mul_fp8(const void *g, int64_t gld, const void *u, int64_t uld, int dtype,
                               const int32_t *live, int N, int I, int scale_kind, uint8_t *q,
                               int64_t qld, float *sq, hipStream_t s) {
  return quant_rows<true>(g, gld, u, uld, dtype, live, N, I, scale_kind, q, qld, sq, s);
}

hipError_t launch_weight_quant_fp8(const void *w, int dtype, int E, int M, int K, int scale_kind,
                                   uint8_t *q, float *scales, hipStream_t s) {
  const unsigned blocks = (unsigned)((int64_t)E * ((M + 127) / 128) * ((K + 127) / 128));
  const int pow2 = scale_kind == AINFER_FP8_SCALE_POW2;
  return enqueue(dtype == AINFER_ACT_F32 ? k_quant_weights<true> : k_quant_weights<false>, blocks, 256,
                 s, w, M, K, pow2, q, scales);
}
