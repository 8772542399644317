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
#include "moe_fp8_parts.h"
#include "moe_gemm_parts.h"

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


// ---- tiles ------------------------------------------------------------------------
// 256 weight rows x NS * 16 rows of x in a workgroup of four waves, each 64 of the weight
// rows: weights go from global memory into registers (no wave shares them), one group
// ahead; rows of x and their scales go through two stages of LDS by DMA, shared by the
// waves.  Two workgroups fit a CU, so that one's waits run under the other's products.
//
// Weight row r of a wave's tile i (four tiles of 16) is row 16 (r / 4) + 4 i + r % 4 of the
// 64, so that a lane ends with 16 neighbouring columns of a row of y.
constexpr int TILE_M = 256;

__device__ const uint8_t fp8_zeros[16] __attribute__((aligned(16))) = {};

template <int NS>
struct Stage {
  static constexpr int X = NS * 16 * 128;           // codes: 128 bytes a row
  static constexpr int SDMA = (NS * 16 + 63) / 64;  // scales, by 64 lanes of 4 bytes each
  static constexpr int BYTES = X + SDMA * 256;
};

// where the rows of each expert's tiles are: tiles before expert e, by 256 threads
struct TileMap {
  int32_t before[1025];
  int32_t part[4];
};

__device__ __forceinline__ void clamp_rows(const Fp8Args &a, int e, int &r0, int &n) {
  r0 = a.offsets ? max(0, min(a.offsets[e], a.N)) : 0;
  n = (a.offsets ? min(a.offsets[e + 1], a.N) : a.N) - r0;
  n = max(n, 0);
}

// tiles of all experts
__device__ __forceinline__ int map_tiles(const Fp8Args &a, int nt, TileMap &map) {
  const int tid = threadIdx.x, wave = tid >> 6;
  int c[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    c[i] = 0;
    if (e < a.E) {
      int r0, n;
      clamp_rows(a, e, r0, n);
      c[i] = (n + nt - 1) / nt;
    }
    mine += c[i];
  }
  const int incl = wave_scan_incl(mine);
  if ((tid & 63) == 63) map.part[wave] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < wave; ++w) at += map.part[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    if (e < a.E) map.before[e] = at;
    at += c[i];
    if (e == a.E - 1) map.before[a.E] = at;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(map.before[a.E]);
}

template <bool F32, int NS>
__device__ __forceinline__ void run_tile(const Fp8Args &a, uint32_t lds0, const uint8_t *lds,
                                         int e, int r0, int n, int m0) {
  using St = Stage<NS>;
  const int tid = tid_opaque(), lane = tid & 63,
            col = lane & 15, qd = lane >> 4;  // per item: nothing is kept across items
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = (a.K + 127) >> 7, groups = (G + 1) & ~1, MB = (a.M + 127) >> 7;
  // weights: a scalar base at the wave's first row, a 32-bit offset for each tile's row
  const int mw = m0 + wave * 64;
  const uint8_t *wbase = a.w + ((int64_t)e * a.M + min(mw, a.M - 1)) * a.K;
  uint32_t woff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * (col >> 2) + 4 * i + (col & 3);
    woff[i] = (uint32_t)max(0, min(r, a.M - 1 - mw)) * (uint32_t)a.K;
  }
  const float *sw = a.scales + ((int64_t)e * MB + min(mw >> 7, MB - 1)) * G;
  // rows of x by DMA: slot s of 16 bytes holds chunk (s & 7) ^ (row & 7) of row s >> 3
  constexpr int DMA = NS * 16 * 8 / 64;  // of 64 lanes each, over four waves
  constexpr int PER = (DMA + 3) / 4;
  const uint64_t xbase = sbase64(a.q + (int64_t)r0 * a.q_ld);
  const uint64_t sbase = sbase64(a.sq + (int64_t)r0 * G);
  uint32_t xoff[PER], xcol[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = (i * 4 + wave) * 64 + lane, row = s >> 3;
    xcol[i] = (uint32_t)(((s & 7) ^ (row & 7)) * 16);
    xoff[i] = (uint32_t)min(row, n - 1) * (uint32_t)a.q_ld;
  }
  // scales of x: place p of the stage's 16 NS floats is row 16 (p % NS) + p / NS
  constexpr int SDMA = St::SDMA;
  uint32_t soff;
  {
    const int p = wave * 64 + lane;
    const int row = 16 * (p % NS) + p / NS;
    soff = (uint32_t)min(row, n - 1) * (uint32_t)G * 4u;
  }
  // Columns behind the row (a last group that is not full, and a last one of an odd number)
  // are zeros in x and any columns of the same row in w: a NaN among those is one of y too.
  auto issue = [&](int g, int stage) __attribute__((always_inline)) {
    const uint32_t base = lds0 + stage * St::BYTES;
    const bool whole = (g + 1) * 128 <= a.K;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (DMA >= 4 * (i + 1) || i * 4 + wave < DMA) {
        const uint32_t to = base + (uint32_t)((i * 4 + wave) * 1024);
        if (whole)
          dma16s(xoff[i] + xcol[i], xbase + (uint64_t)g * 128u, to);
        else
          dma16(g * 128 + xcol[i] < (uint32_t)a.K ? (const uint8_t *)xbase + g * 128 + xoff[i] + xcol[i]
                                                  : fp8_zeros, to);
      }
    }
    if (wave < SDMA) {
      const uint32_t to = base + St::X + (uint32_t)(wave * 256);
      if (g < G) dma4s(soff, sbase + (uint64_t)g * 4u, to);
      else dma4s(0u, (uint64_t)(uintptr_t)fp8_zeros, to);
    }
  };
  auto load_w = [&](int g, Codes (&w)[4]) __attribute__((always_inline)) {
    g = min(g, G - 1);
    const uint8_t *p = wbase + (int64_t)g * 128;
    const uint32_t c0 = g * 128 + qd * 16 < a.K ? qd * 16 : 0;
    const uint32_t c1 = g * 128 + qd * 16 + 64 < a.K ? qd * 16 + 64 : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i].v[0] = *(const u32x4 *)(p + (woff[i] + c0));
      w[i].v[1] = *(const u32x4 *)(p + (woff[i] + c1));
    }
  };
  f32x4 acc[NS][4];
#pragma unroll
  for (int j = 0; j < NS; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t xr0 = (uint32_t)(col * 128 + ((qd ^ (col & 7)) << 4));
  float swv = 0.f;  // lane l: the weights' scale of group 64 (g / 64) + l

  auto step = [&](int g, Codes (&w)[4], Codes (&next)[4]) __attribute__((always_inline)) {
    if ((g & 63) == 0) swv = sw[min(g + lane, G - 1)];
    wait_vm<0>();  // this thread's DMA of group g
    block_barrier();
    if (g + 1 < groups) {
      issue(g + 1, (g + 1) & 1);
      load_w(g + 1, next);
    }
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t *st = lds + (g & 1) * St::BYTES;
    const float s = __uint_as_float(
        __builtin_amdgcn_readlane((int)__float_as_uint(swv), g & 63));
    // One product and the four fmas of the one two before it at a time: the fmas run under
    // the products.  The barriers keep the compiler from reading all rows first (spills).
    Codes x[2];
    float f[2];
    f32x4 d[3];
    auto read_row = [&](int j) {
      x[j & 1] = {{*(const u32x4 *)(st + xr0 + j * 2048), *(const u32x4 *)(st + (xr0 ^ 64) + j * 2048)}};
      f[j & 1] = *(const float *)(st + St::X + (col * NS + j) * 4) * s;
    };
    read_row(0);
#pragma unroll
    for (int t = 0; t < 4 * NS + 2; ++t) {
      const int j = t >> 2, i = t & 3;
      if (t < 4 * NS) d[t % 3] = group_dot<F32>(w[i], x[j & 1]);
      if (t >= 2) {
        const int u = t - 2;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[u >> 2][u & 3][r] = fmaf(f[(u >> 2) & 1], d[u % 3][r], acc[u >> 2][u & 3][r]);
        // no instruction: the sums are due here, not after the next group's branch
        asm volatile("" : "+v"(acc[u >> 2][u & 3]));
      }
      if (i == 1 && j + 1 < NS) read_row(j + 1);  // f of row j - 1 has been used
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  Codes w0[4], w1[4];
  block_barrier();  // the ring's last readers, of the item before
  issue(0, 0);
  load_w(0, w0);
  for (int g = 0; g < groups; g += 2) {
    step(g, w0, w1);
    step(g + 1, w1, w0);
  }

  // 16 neighbouring columns of row 16 j + col
  const int m = mw + 16 * qd;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int row = 16 * j + col;
    if (row < n) {
      const int64_t at = (int64_t)(r0 + row) * a.y_ld + m;
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = acc[j][i >> 2][i & 3];
      if (m + 16 <= a.M) {
        store_row<F32>(a.y, at, v);
      } else {
#pragma unroll
        for (int i = 0; i < 15; ++i)
          if (m + i < a.M) store_one<F32>(a.y, at + i, v[i]);
      }
    }
  }
}

// Items (tile, 256 weight rows) of an expert in bands of 8 tiles, tiles first, so that
// the 64 workgroups of an XCD read few tiles and few weights at a time from its L2.
template <bool F32, int NT>
__global__ __launch_bounds__(256, 2) void k_fp8_tiles(Fp8Args a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * Stage<NT / 16>::BYTES];
  __shared__ TileMap map;
  const int mb = (a.M + TILE_M - 1) / TILE_M;
  const int64_t items = (int64_t)map_tiles(a, NT, map) * mb;
  const int xcd = blockIdx.x % N_XCD, slots = gridDim.x / N_XCD;
  const int64_t end = items * (xcd + 1) / N_XCD;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  for (int64_t it = items * xcd / N_XCD + blockIdx.x / N_XCD; it < end; it += slots) {
    const int tile = (int)(it / mb);
    int lo = 0, hi = a.E;  // the last expert that starts at or before the tile
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (map.before[mid] <= tile) lo = mid;
      else hi = mid;
    }
    const int e = __builtin_amdgcn_readfirstlane(lo);
    int r0, n;
    clamp_rows(a, e, r0, n);
    const int first = __builtin_amdgcn_readfirstlane(map.before[e]);
    const int tiles = (n + NT - 1) / NT;
    const int64_t local = it - (int64_t)first * mb;
    const int band = (int)(local / (8 * mb)), in_band = (int)(local - (int64_t)band * 8 * mb);
    const int wide = min(8, tiles - 8 * band);
    const int t = 8 * band + in_band % wide, m0 = in_band / wide * TILE_M;
    r0 = __builtin_amdgcn_readfirstlane(r0 + t * NT);
    n = __builtin_amdgcn_readfirstlane(min(NT, n - t * NT));
    const int ns = (n + 15) / 16;
    if constexpr (NT > 64) {
      if (ns > 6) run_tile<F32, 8>(a, lds0, lds, e, r0, n, m0);
      else if (ns > 4) run_tile<F32, 6>(a, lds0, lds, e, r0, n, m0);
    }
    if (ns <= 4) {
      if (ns > 2) run_tile<F32, 4>(a, lds0, lds, e, r0, n, m0);
      else if (ns == 2) run_tile<F32, 2>(a, lds0, lds, e, r0, n, m0);
      else run_tile<F32, 1>(a, lds0, lds, e, r0, n, m0);
    }
  }
}

}  // namespace

hipError_t launch_fp8_product(const Fp8Args &a, int y_dtype, hipStream_t s) {
  const bool f32 = y_dtype == AINFER_ACT_F32;
  if (a.N > 8 * a.E) {
    const int nt = f32 ? 64 : 128;
    const int64_t most = (int64_t)(a.N / nt + std::min(a.E, a.N)) * ((a.M + TILE_M - 1) / TILE_M);
    const int grid = (int)std::min<int64_t>(512, (most + N_XCD - 1) / N_XCD * N_XCD);
    if (f32) k_fp8_tiles<true, 64><<<grid, 256, 0, s>>>(a);
    else k_fp8_tiles<false, 128><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
  }
  // at most: full tiles, and one that is not full for each expert
  const int64_t tiles = a.offsets ? a.N / 16 + std::min(a.E, a.N) : (a.N + 15) / 16;
  const int64_t items = tiles * ((a.M + 15) / 16);
  const int grid = (int)std::min<int64_t>(items, 1 << 20);
  if (f32)
    k_fp8_rows<true><<<grid, 256, 0, s>>>(a, items);
  else
    k_fp8_rows<false><<<grid, 256, 0, s>>>(a, items);
  return hipGetLastError();
}
