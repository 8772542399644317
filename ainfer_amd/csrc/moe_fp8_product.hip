// moe_fp8_product.hip - y = x W^T with e4m3 codes and a scale for every 128 columns of
// x and every 128 x 128 block of W, for one matrix or for rows sorted by expert
// (ainfer_moe_fp8_product).
//
// v_mfma_f32_16x16x128_f8f6f4 takes exactly one scale group of 16 weight rows and 16
// rows of x, so a group's dot comes out whole and enters the fp32 sum as
// fma(s_x s_w, dot, sum).  Weights are its first operand: a lane's four results are
// four neighbouring columns of one row of y, with one scale for all four.
#include <algorithm>

#include "moe_common.h"
#include "moe_internal.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Two 16-byte chunks of codes of a row, as the lanes hold a group: lane (row l % 16,
// quarter l / 16) columns [16 quarter, +16) and [64 + 16 quarter, +16).
struct Codes {
  u32x4 v[2];
};

// The group's dot of 16 x 16 rows, fp32 out.
//
// v_mfma_f32_16x16x128_f8f6f4 aligns every eight neighbouring products to the largest
// one and drops what is more than 13 bits below it (measured; the other fp8 MFMAs do the
// same).  That is 1.4e-5 of a sum of normal values, far below a bf16 output's rounding,
// and at most 7 * 2^-13 of the sum of magnitudes.  An fp32 output is to be nearer: its
// codes become fp16 values (exact) for v_mfma_f32_16x16x32_f16, which is off by 1e-8, at
// half the matrix rate and 32 conversions a lane.
__device__ __forceinline__ f16x8 to_f16(uint32_t a, uint32_t b) {
  const f16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true)};
  return f16x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}
template <bool F32>
__device__ __forceinline__ f32x4 group_dot(const Codes &a, const Codes &b) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
  if constexpr (F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(to_f16(a.v[h][i], a.v[h][i + 1]),
                                                   to_f16(b.v[h][i], b.v[h][i + 1]), d, 0, 0, 0);
    return d;
  } else {
    const i32x8 av = {(int)a.v[0][0], (int)a.v[0][1], (int)a.v[0][2], (int)a.v[0][3],
                      (int)a.v[1][0], (int)a.v[1][1], (int)a.v[1][2], (int)a.v[1][3]};
    const i32x8 bv = {(int)b.v[0][0], (int)b.v[0][1], (int)b.v[0][2], (int)b.v[0][3],
                      (int)b.v[1][0], (int)b.v[1][1], (int)b.v[1][2], (int)b.v[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, d, 0, 0, 0, 0, 0, 0);
  }
}

struct Tile {
  int e, r0, n;  // expert, first row, rows; n = 0: none
};

// Tile `tile` of NT rows, in the order of the experts' rows.  offsets (what the caller
// gives) are taken as rows of [0, N), whatever they hold.  256 threads, E <= 1024.
template <int NT>
__device__ __forceinline__ Tile find_tile(const int32_t *offsets, int E, int N, int64_t tile) {
  __shared__ Tile found;
  __shared__ int32_t part[4];
  if (!offsets) {
    const int64_t r0 = tile * NT;
    return Tile{0, (int)r0, (int)min((int64_t)NT, max((int64_t)0, N - r0))};
  }
  const int tid = threadIdx.x, wave = tid >> 6;
  int start[4], rows[4], tiles = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = min(tid * 4 + i, E - 1);
    start[i] = max(0, min(offsets[e], N));
    rows[i] = tid * 4 + i < E ? max(0, min(offsets[e + 1], N) - start[i]) : 0;
    tiles += (rows[i] + NT - 1) / NT;
  }
  const int incl = wave_scan_incl(tiles);
  __syncthreads();  // the last call's readers of found and part
  if (tid == 0) found = Tile{0, 0, 0};
  if ((tid & 63) == 63) part[wave] = incl;
  __syncthreads();
  int64_t at = tile - (incl - tiles);
  for (int w = 0; w < wave; ++w) at -= part[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (rows[i] + NT - 1) / NT;
    if (at >= 0 && at < c)
      found = Tile{tid * 4 + i, start[i] + (int)at * NT, min(NT, rows[i] - (int)at * NT)};
    at -= c;
  }
  __syncthreads();
  return found;
}

// 16 bytes of codes, none behind the row's K columns
__device__ __forceinline__ u32x4 codes_at(const uint8_t *row, int col, int K) {
  return col < K ? *(const u32x4 *)(row + col) : u32x4{0, 0, 0, 0};
}

// 16 weight rows x at most 16 rows of x: four waves take every fourth group of 128
// columns, and their sums are added in the waves' order.
template <bool F32>
__global__ __launch_bounds__(256) void k_fp8_rows(Fp8Args a, int64_t items) {
  __shared__ f32x4 sums[4][64];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, qd = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slabs = (a.M + 15) / 16, G = (a.K + 127) / 128, MB = (a.M + 127) / 128;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const Tile t = find_tile<16>(a.offsets, a.E, a.N, it / slabs);
    if (t.n == 0) return;  // no tile from here on
    const int m0 = (int)(it % slabs) * 16;
    const uint8_t *wr = a.w + ((int64_t)t.e * a.M + min(m0 + c, a.M - 1)) * a.K;
    const float *sw = a.scales + ((int64_t)t.e * MB + m0 / 128) * G;
    const int64_t row = t.r0 + min(c, t.n - 1);
    const uint8_t *xr = a.q + row * a.q_ld;
    const float *sx = a.sq + row * G;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int g = wave; g < G; g += 4) {
      const int col = g * 128 + qd * 16;
      const Codes wv = {{codes_at(wr, col, a.K), codes_at(wr, col + 64, a.K)}};
      const Codes xv = {{codes_at(xr, col, a.K), codes_at(xr, col + 64, a.K)}};
      const f32x4 dot = group_dot<F32>(wv, xv);
      const float s = sx[g] * sw[g];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(s, dot[i], acc[i]);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < t.n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + 4 * qd + i;
        const float v = (sums[0][lane][i] + sums[1][lane][i]) + (sums[2][lane][i] + sums[3][lane][i]);
        if (m < a.M) {
          const int64_t at = row * a.y_ld + m;
          if constexpr (F32) ((float *)a.y)[at] = v;
          else ((uint16_t *)a.y)[at] = f32_to_bf16(v);
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_fp8_product(const Fp8Args &a, int y_dtype, hipStream_t s) {
  // at most: full tiles, and one that is not full for each expert
  const int64_t tiles = a.offsets ? a.N / 16 + std::min(a.E, a.N) : (a.N + 15) / 16;
  const int64_t items = tiles * ((a.M + 15) / 16);
  const int grid = (int)std::min<int64_t>(items, 1 << 20);
  if (y_dtype == AINFER_ACT_F32)
    k_fp8_rows<true><<<grid, 256, 0, s>>>(a, items);
  else
    k_fp8_rows<false><<<grid, 256, 0, s>>>(a, items);
  return hipGetLastError();
}
