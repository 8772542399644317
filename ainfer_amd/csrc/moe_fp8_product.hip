// moe_fp8_product.hip - y = x W^T with e4m3 codes and a scale for every 128 columns of
// x and every 128 x 128 block of W, for one matrix or for rows sorted by expert
// (ainfer_moe_fp8_product).
//
// v_mfma_f32_16x16x128_f8f6f4 takes exactly one scale group of 16 weight rows and 16
// rows of x, so a group's dot comes out whole and enters the fp32 sum as
// fma(s_x s_w, dot, sum).  Weights are its first operand: a lane's four results are
// four neighbouring columns of one row of y, with one scale for all four.
//
// Weights are laid out once (ainfer_moe_fp8_pack) as this instruction takes them: 64 rows x
// 128 columns are four tiles of 16 rows, each 2 KB in the order of the lanes, so that a wave's
// load is 1 KB of neighbouring bytes.  (Read from plain rows, 16 neighbouring lanes touch 16
// rows, which the CU's address unit takes one by one: 8192^3 ran at 1394 TFLOP/s.)  Row r of tile
// i is row 32 (i / 2) + 8 (r / 4) + 4 (i % 2) + r % 4 of the 64, so that the lane that holds four
// results of each tile holds two times 8 neighbouring columns of a row of y, and the four lanes of
// a row 32.  Rows and columns behind the matrix are zeros.
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
// v_mfma_f32_16x16x128_f8f6f4 aligns every eight neighbouring products to the largest sum of
// two codes' exponents and cuts what is more than 13 bits below it towards zero (measured; the
// other fp8 MFMAs do the same).  That is 1.1e-5 of a group's sum of normal values, far below a
// bf16 output's rounding: products of 4096 columns are as far from the 64-bit ones as the
// rounded 64-bit ones are (1.657e-3 of the norm; 1.2% of the values are the neighbour).  At most
// it is 7 * 2^-13 of the sum of magnitudes, and 8 times that beside subnormal codes, whose exponent is
// 2^-6's whatever their value.  An fp32 output is to be nearer: its codes become fp16 values (exact)
// for v_mfma_f32_16x16x32_f16, which is off by 1e-8, at half the matrix rate and 32 conversions a
// lane.
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

// the packed tile i of rows 64 mb .. +63 and group g
__device__ __forceinline__ const uint8_t *tile_at(const Fp8Args &a, int e, int mb, int g, int i) {
  const int G = (a.K + 127) >> 7, MB64 = (a.M + 63) >> 6;
  return a.w + (((int64_t)e * MB64 + mb) * G + g) * 8192 + i * 2048;
}

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

// the last expert that starts at or before the tile: the one that holds it
__device__ __forceinline__ int expert_of_tile(const TileMap &map, int E, int tile) {
  int lo = 0, hi = E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (map.before[mid] <= tile) lo = mid;
    else hi = mid;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Lane l's 16 or 4 bytes at `off` of the buffer to the wave's LDS address + 16 l or 4 l (zeros
// where off is behind the buffer).  The compiler counts the copy among the loads in flight but
// is not told what it writes, so that it waits for none of them before a read of the ring:
// step() does.  (A global_load_lds would do that too, but counts as an access of both
// memories, for which the compiler waits until nothing is in flight.)
typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ void dma_x4(__amdgpu_buffer_rsrc_t b, uint32_t off, uint32_t to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_void *)(uintptr_t)to, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void dma_x1(__amdgpu_buffer_rsrc_t b, uint32_t off, uint32_t to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_void *)(uintptr_t)to, 4, off, 0, 0, 0);
}

// ---- split ------------------------------------------------------------------------
// 16 R weight rows x 16 NS rows of x in a workgroup of four waves that take every fourth
// group of 128 columns each; their sums are added in the waves' order.  For calls with too few
// 256-row tiles to fill the CUs.  One row is bound by the weights: 5120 -> 17408 17.5 us, 5.1
// TB/s.  Each wave copies its own rows of x into LDS of its own
// (no barriers), three stages, two groups ahead, and loads its weights into registers.
template <int NS>
struct Share {
  static constexpr int X = NS * 2048;
  static constexpr int BYTES = X + 256;  // a stage of one wave: codes, scales
};

template <bool F32, int R, int NS>
__global__ __launch_bounds__(256) void k_fp8_split(Fp8Args a) {
  using Sh = Share<NS>;
  constexpr int RING = 4 * 3 * Sh::BYTES, SUMS = 3 * R * NS * 1024;
  __shared__ __attribute__((aligned(16))) uint8_t lds[RING > SUMS ? RING : SUMS];
  __shared__ TileMap map;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, qd = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slabs = (a.M + 63) / 64 * (4 / R), G = (a.K + 127) >> 7, MB = (a.M + 127) >> 7;
  const uint8_t *mine = lds + wave * 3 * Sh::BYTES;
  const uint32_t mine0 = (uint32_t)(uintptr_t)lds + (uint32_t)(wave * 3 * Sh::BYTES);
  const int64_t items = (int64_t)map_tiles(a, 16 * NS, map) * slabs;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int tile = (int)(it / slabs), e = expert_of_tile(map, a.E, tile);
    int r0, n;
    clamp_rows(a, e, r0, n);
    const int before = __builtin_amdgcn_readfirstlane(tile - map.before[e]) * 16 * NS;
    r0 = __builtin_amdgcn_readfirstlane(r0 + before);
    n = __builtin_amdgcn_readfirstlane(min(16 * NS, n - before));
    const int slab = (int)(it % slabs), mb = slab / (4 / R), i0 = slab % (4 / R) * R;
    const uint8_t *wbase = tile_at(a, e, mb, 0, i0) + lane * 16;
    int zero = 0;  // opaque: a vector load is in the counts below, a scalar one would not be
    asm volatile("" : "+v"(zero));
    const float *sw = a.scales + ((int64_t)e * MB + (mb >> 1)) * G + zero;
    const __amdgpu_buffer_rsrc_t xbuf =
        make_rsrc(a.q + (int64_t)r0 * a.q_ld, (uint32_t)(n - 1) * (uint32_t)a.q_ld + (uint32_t)a.K);
    const __amdgpu_buffer_rsrc_t sbuf = make_rsrc(a.sq + (int64_t)r0 * G, (uint32_t)(n * G) * 4u);
    // as in the tiles: chunk (s & 7) ^ (row & 7) of row s >> 3 in slot s
    uint32_t xoff[2 * NS];
    const uint32_t xcol = (uint32_t)(((lane & 7) ^ (lane >> 3)) * 16);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i)
      xoff[i] = (uint32_t)min(8 * i + (lane >> 3), n - 1) * (uint32_t)a.q_ld + xcol;
    const uint32_t soff = (uint32_t)min(16 * (lane % NS) + lane / NS, n - 1) * (uint32_t)G * 4u;
    struct Group {
      Codes w[R];
      float s;
    };
    const int mineG = (G - wave + 3) / 4;  // groups wave, wave + 4, ...
    auto issue = [&](int u, int stage, Group &next) __attribute__((always_inline)) {
      const int g = wave + 4 * u;
      const bool past = g * 128 + xcol >= (uint32_t)a.K;
      const uint32_t to = mine0 + (uint32_t)(stage * Sh::BYTES);
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i)
        dma_x4(xbuf, past ? BUF_OOB : xoff[i] + g * 128, to + (uint32_t)(i * 1024));
      dma_x1(sbuf, soff + g * 4, to + Sh::X);
      // the loads of weights stay behind the copies: step() counts on it
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      next.s = sw[g];
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          next.w[i].v[h] = __builtin_nontemporal_load(
              (const u32x4 *)(wbase + (int64_t)g * 8192 + i * 2048 + h * 1024));
      __builtin_amdgcn_sched_barrier(0);
    };
    f32x4 acc[NS][R];
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int i = 0; i < R; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint32_t xr0 = (uint32_t)(col * 128 + ((qd ^ (col & 7)) << 4));
    // the wave's group u, in a stage; behind its DMA there are its own 2 R + 1 loads and all
    // of the next group's
    auto step = [&](int u, int stage, Group &c, auto loads, int fill, Group &next)
                    __attribute__((always_inline)) {
      constexpr bool LOADS = decltype(loads)::value;
      if constexpr (LOADS) {
        wait_vm<2 * (2 * R + 1) + 2 * NS + 1>();
        issue(min(u + 2, mineG - 1), fill, next);
      } else {
        wait_vm<0>();
      }
      const uint8_t *st = mine + stage * Sh::BYTES;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const Codes x = {{*(const u32x4 *)(st + xr0 + j * 2048), *(const u32x4 *)(st + (xr0 ^ 64) + j * 2048)}};
        const float f = *(const float *)(st + Sh::X + (col * NS + j) * 4) * c.s;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const f32x4 d = group_dot<F32>(c.w[i], x);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(f, d[r], acc[j][i][r]);
        }
      }
      // the stage has been read before it is filled again
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    Group c0, c1, c2;
    if (mineG > 0) {
      issue(0, 0, c0);
      issue(min(1, mineG - 1), 1, c1);
    }
    int u = 0;
    for (; u + 3 <= mineG; u += 3) {
      step(u, 0, c0, std::true_type(), 2, c2);
      step(u + 1, 1, c1, std::true_type(), 0, c0);
      step(u + 2, 2, c2, std::true_type(), 1, c1);
    }
    if (u < mineG) {
      step(u, 0, c0, std::false_type(), 2, c2);
      if (u + 1 < mineG) step(u + 1, 1, c1, std::false_type(), 0, c0);
    }
    wait_vm<0>();  // no copy into the ring is in flight
    __syncthreads();
    f32x4 *sums = (f32x4 *)lds;
    if (wave > 0) {
#pragma unroll
      for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int i = 0; i < R; ++i) sums[((wave - 1) * NS * R + j * R + i) * 64 + lane] = acc[j][i];
    }
    __syncthreads();
    if (wave == 0) {
      const int m = mb * 64 + 8 * qd;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        if (16 * j + col >= n) continue;
        const int64_t at = (int64_t)(r0 + 16 * j + col) * a.y_ld;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int c = m + 32 * ((i0 + i) >> 1) + 4 * ((i0 + i) & 1);
          f32x4 v = acc[j][i];
#pragma unroll
          for (int w = 0; w < 3; ++w) v += sums[(w * NS * R + j * R + i) * 64 + lane];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c + r < a.M) store_one<F32>(a.y, at + c + r, v[r]);
        }
      }
    }
    __syncthreads();
  }
}

// ---- tiles ------------------------------------------------------------------------
// 256 weight rows x NS * 16 rows of x in a workgroup of four waves, each 64 of the weight
// rows: weights go from global memory into registers (no wave shares them); rows of x and
// their scales go through three stages of LDS by DMA, shared by the waves, two groups ahead;
// weights AHEAD groups and the time from their last use to the next step.  Two workgroups fit a
// CU, so that one's waits run under the other's products.  (One workgroup of eight waves with
// 256 x 192: 8192^3 637 instead of 580 us.)
//
// Bound by the loads' way through a CU's L1: a group of 256 x 128 is 48 KB for 128 products, and
// 8192^3 brings 50 bytes a ns to each CU (without the loads the products alone run at 2622
// TFLOP/s).  8192^3 507 us, 2170 TFLOP/s (a library's bf16 product 1366); 4096 x 5120 -> 17408
// 354, 2065; 64 experts of about 512 rows, 4096 -> 2048 335 to 351, 1570 to 1640: there the weights
// come from memory, not from a cache; with fp32 outputs 8192 x 4096 -> 4096 263, 1047.
constexpr int TILE_M = 256;

template <int NS>
struct Stage {
  static constexpr int DMA = (NS + 1) / 2;          // 16-byte copies a lane, of four waves
  static constexpr int X = DMA * 4096;              // codes: 128 bytes a row
  static constexpr int BYTES = X + 1024;            // scales: one a lane
};

template <bool F32, int NS, int AHEAD>
__device__ __forceinline__ void run_tile(const Fp8Args &a, uint32_t lds0, const uint8_t *lds,
                                         int e, int r0, int n, int m0) {
  using St = Stage<NS>;
  const int tid = tid_opaque(), lane = tid & 63,
            col = lane & 15, qd = lane >> 4;  // per item: nothing is kept across items
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = (a.K + 127) >> 7, MB = (a.M + 127) >> 7;
  int zero = 0;  // opaque: a vector load is in the counts below, a scalar one would not be
  asm volatile("" : "+v"(zero));
  const int mw = m0 + wave * 64, mbw = min(mw >> 6, ((a.M + 63) >> 6) - 1);
  const uint8_t *wbase = tile_at(a, e, mbw, 0, 2);
  const float *sw = a.scales + ((int64_t)e * MB + (mbw >> 1)) * G;
  // rows of x by DMA: slot s of 16 bytes holds chunk (s & 7) ^ (row & 7) of row s >> 3
  const __amdgpu_buffer_rsrc_t xbuf =
      make_rsrc(a.q + (int64_t)r0 * a.q_ld, (uint32_t)(n - 1) * (uint32_t)a.q_ld + (uint32_t)a.K);
  const __amdgpu_buffer_rsrc_t sbuf = make_rsrc(a.sq + (int64_t)r0 * G, (uint32_t)(n * G) * 4u);
  uint32_t xoff[St::DMA];
  const uint32_t xcol = (uint32_t)(((lane & 7) ^ (lane >> 3)) * 16);
#pragma unroll
  for (int i = 0; i < St::DMA; ++i)
    xoff[i] = (uint32_t)min((i * 4 + wave) * 8 + (lane >> 3), n - 1) * (uint32_t)a.q_ld + xcol;
  // scales: place p of the stage's is row 16 (p % NS) + p / NS
  const int sp = wave * 64 + lane;
  const uint32_t soff = (uint32_t)min(16 * (sp % NS) + sp / NS, n - 1) * (uint32_t)G * 4u;
  auto issue = [&](int g, uint32_t stage) __attribute__((always_inline)) {
    const bool past = g * 128 + xcol >= (uint32_t)a.K;
#pragma unroll
    for (int i = 0; i < St::DMA; ++i)
      dma_x4(xbuf, past ? BUF_OOB : xoff[i] + g * 128, stage + (uint32_t)((i * 4 + wave) * 1024));
    dma_x1(sbuf, soff + g * 4, stage + St::X + (uint32_t)(wave * 256));
    // the loads of weights stay behind the copies: step() counts on it
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  const uint32_t wlane = (uint32_t)lane * 16u;
  auto load_s = [&](int g) __attribute__((always_inline)) { return sw[g + zero]; };
  auto load_w = [&](int g, int i, Codes &w) __attribute__((always_inline)) {
    const uint8_t *p = wbase + (int64_t)g * 8192;
#pragma unroll
    for (int h = 0; h < 2; ++h) w.v[h] = *(const u32x4 *)(p + wlane + ((i - 2) * 2048 + h * 1024));
  };
  struct Weights {
    Codes w[4];
    float s;
  };
  auto load_all = [&](int g, Weights &w) __attribute__((always_inline)) {
    w.s = load_s(g);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_w(g, i, w.w[i]);
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4 acc[NS][4];
#pragma unroll
  for (int j = 0; j < NS; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t xr0 = (uint32_t)(col * 128 + ((qd ^ (col & 7)) << 4));
  const uint32_t xs0 = (uint32_t)(St::X + col * NS * 4);

  // Group g: its rows were sent for at the start of the step two before, its weights at the end
  // of the one AHEAD + 1 before, as their registers came free.  (Rows, then weights, at the
  // start of the step AHEAD before: 8192^3 543 instead of 507 us, 64 experts of 512 rows 375
  // instead of 346, 1024 x 4096 -> 4096 37.6 instead of 32.9.)  Behind the copies of g there are
  // the loads of one group's weights, the copies of g + 1 and another group's weights.  The
  // loop's last steps load the last group again, so that this count is the same in every one of
  // them.  (A load whose value nothing takes would not be there to be counted: the steps behind
  // the loop issue none, and wait for what is left.)
  constexpr int NEWER = 9 + St::DMA + 1 + 9;
  uint32_t here = 0, fill = 2 * St::BYTES;  // the stages of groups g and g + 2
  auto step = [&](int g, Weights &w, auto loads) __attribute__((always_inline)) {
    constexpr bool LOADS = decltype(loads)::value;
    if constexpr (LOADS) wait_vm<NEWER>();
    else wait_vm<0>();
    block_barrier();
    if constexpr (LOADS) issue(min(g + 2, G - 1), lds0 + fill);
    const int next = min(g + AHEAD + 1, G - 1);
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t *st = lds + here;
    here = here == 2 * St::BYTES ? 0 : here + St::BYTES;
    fill = fill == 2 * St::BYTES ? 0 : fill + St::BYTES;
    // One product and the four fmas of the one two before it at a time: the fmas run under
    // the products.  The barriers keep the compiler from reading all rows first (spills).
    constexpr int XB = F32 ? 1 : 2;  // fp32: the registers are the conversions'
    Codes x[XB];
    float f[2];
    f32x4 d[3];
    auto read_row = [&](int j) {
      x[j % XB] = {{*(const u32x4 *)(st + xr0 + j * 2048), *(const u32x4 *)(st + (xr0 ^ 64) + j * 2048)}};
      f[j & 1] = *(const float *)(st + xs0 + j * 4) * w.s;
    };
    read_row(0);
#pragma unroll
    for (int t = 0; t < 4 * NS + 2; ++t) {
      const int j = t >> 2, i = t & 3;
      if (t < 4 * NS) d[t % 3] = group_dot<F32>(w.w[i], x[j % XB]);
      if (t >= 2) {
        const int u = t - 2;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[u >> 2][u & 3][r] = fmaf(f[(u >> 2) & 1], d[u % 3][r], acc[u >> 2][u & 3][r]);
        // no instruction: the sums are due here, not after the next group's branch
        asm volatile("" : "+v"(acc[u >> 2][u & 3]));
      }
      // (f of row j - 1 has been used)
      if (i == (XB == 2 ? 1 : 3) && j + 1 < NS) read_row(j + 1);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (LOADS) {
        if (j == NS - 1) {
          if (i == 0) w.s = load_s(next);
          load_w(next, i, w.w[i]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  // (loops without breaks, for which the compiler would wait for every load)
  using yes = std::true_type;
  using no = std::false_type;
  Weights w0, w1, w2;
  // the ring's last readers and copies, of the item before
  wait_vm<0>();
  block_barrier();
  if constexpr (AHEAD > 1) load_all(0, w0);
  issue(0, lds0);
  load_all(min(AHEAD - 1, G - 1), AHEAD > 1 ? w1 : w0);
  issue(min(1, G - 1), lds0 + St::BYTES);
  load_all(min(AHEAD, G - 1), AHEAD > 1 ? w2 : w1);
  int g = 0;
  if constexpr (AHEAD > 1) {
    for (; g + 3 <= G; g += 3) {
      step(g, w0, yes());
      step(g + 1, w1, yes());
      step(g + 2, w2, yes());
    }
    if (g < G) {
      step(g, w0, no());
      if (g + 1 < G) step(g + 1, w1, no());
    }
  } else {
    for (; g + 2 <= G; g += 2) {
      step(g, w0, yes());
      step(g + 1, w1, yes());
    }
    if (g < G) step(g, w0, no());
  }

  // Row 16 j + col, two times 32 columns: the row's four lanes write 64 neighbouring bytes at a
  // time, bf16 as they hold them (8 columns each), fp32 after their two pieces of 4 columns
  // became pieces qd and 4 + qd of the 32.  (16 columns a lane, written in pieces 64 bytes
  // apart: 1024 x 1024 -> 16384 with fp32 outputs 53.7 instead of 44.5 us.)
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int row = 16 * j + col;
    const int64_t at = (int64_t)(r0 + row) * a.y_ld;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 v[2] = {acc[j][2 * h], acc[j][2 * h + 1]};
      if constexpr (F32) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0][d]),
                                                           __float_as_uint(v[1][d]), false, false);
          const u32x2 t = __builtin_amdgcn_permlane32_swap(s[0], s[1], false, false);
          v[0][d] = __uint_as_float(t[0]);
          v[1][d] = __uint_as_float(t[1]);
        }
        if (row >= n) continue;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int m = mw + 32 * h + 16 * b + 4 * qd;
          if (m + 4 <= a.M) {
            *(f32x4_any *)((float *)a.y + at + m) = v[b];
          } else {
#pragma unroll
            for (int d = 0; d < 3; ++d)
              if (m + d < a.M) ((float *)a.y)[at + m + d] = v[b][d];
          }
        }
      } else if (row < n) {
        const int m = mw + 32 * h + 8 * qd;
        const float x[8] = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]};
        if (m + 8 <= a.M) {
          store_row<false>(a.y, at + m, x);
        } else {
#pragma unroll
          for (int d = 0; d < 7; ++d)
            if (m + d < a.M) store_one<false>(a.y, at + m + d, x[d]);
        }
      }
    }
  }
}

// Items (tile, 256 weight rows) of an expert in bands of 8 tiles, tiles first, so that
// the 64 workgroups of an XCD read few tiles and few weights at a time from its L2.
template <bool F32, int NT, int AHEAD>
__global__ __launch_bounds__(256, 2) void k_fp8_tiles(Fp8Args a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[3 * Stage<NT / 16>::BYTES];
  __shared__ TileMap map;
  const int mb = (a.M + TILE_M - 1) / TILE_M;
  const int64_t items = (int64_t)map_tiles(a, NT, map) * mb;
  const int xcd = blockIdx.x % N_XCD, slots = gridDim.x / N_XCD;
  const int64_t end = items * (xcd + 1) / N_XCD;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  for (int64_t it = items * xcd / N_XCD + blockIdx.x / N_XCD; it < end; it += slots) {
    const int tile = (int)(it / mb);
    const int e = expert_of_tile(map, a.E, tile);
    int r0, n;
    clamp_rows(a, e, r0, n);
    const int first = __builtin_amdgcn_readfirstlane(map.before[e]);
    const int tiles = (n + NT - 1) / NT;
    const int64_t local = it - (int64_t)first * mb;
    const int band = (int)(local / (8 * mb)), in_band = (int)(local - (int64_t)band * 8 * mb);
    const int wide = min(8, tiles - 8 * band);
    const int t = 8 * band + in_band % wide, m0 = in_band / wide * TILE_M;
    // the expert's 16s of rows shared evenly by its tiles
    const int units = (n + 15) / 16;
    const int u0 = (int)((int64_t)units * t / tiles), ns = (int)((int64_t)units * (t + 1) / tiles) - u0;
    r0 = __builtin_amdgcn_readfirstlane(r0 + 16 * u0);
    n = __builtin_amdgcn_readfirstlane(min(16 * ns, n - 16 * u0));
    auto run = [&](auto ns_c) {
      constexpr int NS = decltype(ns_c)::value;
      if constexpr (NS * 16 <= NT) run_tile<F32, NS, AHEAD>(a, lds0, lds, e, r0, n, m0);
    };
    switch (__builtin_amdgcn_readfirstlane(ns)) {
    case 1: run(std::integral_constant<int, 1>()); break;
    case 2: run(std::integral_constant<int, 2>()); break;
    case 3: run(std::integral_constant<int, 3>()); break;
    case 4: run(std::integral_constant<int, 4>()); break;
    case 5: run(std::integral_constant<int, 5>()); break;
    case 6: run(std::integral_constant<int, 6>()); break;
    case 7: run(std::integral_constant<int, 7>()); break;
    case 8: run(std::integral_constant<int, 8>()); break;
    }
  }
  wait_vm<0>();  // no copy into this workgroup's LDS outlives it
}

}  // namespace

Fp8Form fp8_form(int E, int M, int K, int N, bool f32) {
  const int nt = f32 ? 64 : 96, G = (K + 127) / 128;
  // what the host knows: at most `used` experts with rows, `each` rows of one on average
  const int64_t used = std::min(E, N), each = N / used;
  const int64_t slabs = (M + 63) / 64, mb = (M + TILE_M - 1) / TILE_M;
  auto row_tiles = [&](int rows) { return std::max<int64_t>(used, (N + rows - 1) / rows); };
  // Tiles or split.  A tile's workgroup takes its K groups one by one, 0.5 us and 0.06 for each
  // 16 rows of x (latency) while its CU is not full; the split form's items take 1 / 1000 us for
  // a group and 64 weight rows x 32 rows of x, and weights that are read for the first time as
  // much and a third again.  So few items of many rows are split (us, bf16; rows x K -> M):
  //   256 x 4096 -> 4096 21.8 split, 29.0 tiles; 384 x 4096 -> 4096 29.9, 29.4; 512 38.5, 29.5;
  //   64 x 5120 -> 17408 44.0, 38.8; 4 experts of 32 rows, 4096 -> 4096 24.2, 20.2; 16 of 18, 2048 ->
  //   2048 21.0, 14.8; 64 of 32, 4096 -> 2048 145, 102; fp32: 4 of 64, 4096 -> 4096 32.6, 37.6;
  //   16 of 18, 2048 -> 2048 20.9, 18.4.
  // With few rows an expert both read weights at the speed of the memory, and the split form
  // gets more of it: 128 rows over 256 experts, 2048 -> 1024 37.6, 41.8; 512 over 512 112, 119; 16
  // experts of 4, 4096 -> 2048 23.6, 29.6; 64 of 8 88.6, 96.3; but with short rows 256 of 7, 2048 ->
  // 1024 108, 97; 64 of 6, 512 -> 4096 42, 31.
  // The average is all that the host knows.  Where N is more than the rows in use, `each` is too
  // high (64 experts, 4096 -> 2048, 512 rows in use: 95 as of N = 4096, 87 split); a caller that
  // knows a smaller bound passes that as N.  Where few experts have most of the rows, the split
  // form reads their weights again for every 16: 90% of 4000 rows on 8 of 512 experts, 4096 ->
  // 2048 799 instead of 580 with tiles (spread evenly 719, 717); of 8192 on 8 of 1024, 4096 ->
  // 1024 785, 610 (706, 723).
  const int64_t items2 = row_tiles(32) * slabs, tile_items = row_tiles(nt) * mb;
  const int64_t units = (each + 15) / 16, per = (units + nt / 16 - 1) / (nt / 16);
  const int64_t ns = (units + per - 1) / per;
  const int64_t few = (f32 ? 1030 + 30 * ns : 440 + 50 * ns) * std::max<int64_t>(512, tile_items) / 512;
  if (items2 + used * slabs * 4 / 3 > few && (each > 12 || (each > 4 && G < 32))) {
    // Higher tiles bring fewer bytes for a product through the CU's L1, which bounds large
    // calls, and leave registers for one group of weights ahead instead of two, which costs calls
    // that do not fill the CUs or bring mostly weights.  us, 96 rows with two groups ahead and 128
    // with one: 4096 x 4096 -> 4096 76, 68; 2048 46.5, 42.9; 1500 x 2048 -> 5000 28.2, 25.3; 64
    // experts of 128 rows, 4096 -> 2048 148, 139; 1024 x 4096 -> 4096 30.9, 38.1; 256 x 5120 -> 17408
    // 40.5, 50.9; 512 experts of 8 rows, 2048 -> 1024 246, 253.  fp32, 64 rows and
    // two ahead, 96 and one: 64 experts of 256 rows, 4096 -> 2048 324, 310; of 128 195, 190; 1119 x
    // 976 -> 13696 45.6, 43.3; 8192 x 4096 -> 4096 271, 267; 2048 x 4096 -> 4096 66, 80; 32 experts of
    // 156, 1024 -> 2048 39, 44.  An expert of up to 64 rows is one tile of either, one of 65 to 96
    // two of 64 or one of 96: experts of 48 rows on average 134, 140 (128 experts, 2048 -> 2048), 103,
    // 108 (96, 2560 -> 1792); 62 114, 114 (96); 64 138, 139 (128), 119, 113 (96), 75, 76 (64, 1024 ->
    // 4096); 72 147, 144 (128), 122, 117 (96), 79, 76 (64); 96 166, 162 (128), 143, 131 (96).
    if (f32 && row_tiles(96) * mb >= 600 && each > 64) return {TILE_M, 96};
    if (f32) return {TILE_M, 64};
    if (row_tiles(128) * mb >= 200 && each > 16) return {TILE_M, 128};
    return {TILE_M, 96};
  }
  // Larger items read less, smaller ones are more: 16 weight rows for a single tile of rows
  // (1 x 5120 -> 17408 17.5, 19.2 with 32); tiles of 32 rows from 128 items of them on
  // (32 x 4096 -> 4096 9.0 with 16, 10.5; 64 x 4096 -> 4096 12.2, 10.3), 64 weight rows
  // from 256 on (64 x 4096 -> 4096 10.3 with 32, 13.5; 128 x 4096 -> 4096 15.8, 13.2).
  if (each > 16 && items2 >= 256) return {64, 32};
  if (each > 16 && items2 >= 128) return {32, 32};
  if (row_tiles(16) > 1) return {32, 16};
  return {16, 16};
}

hipError_t launch_fp8_product(const Fp8Args &a, int y_dtype, hipStream_t s) {
  const bool f32 = y_dtype == AINFER_ACT_F32;
  const Fp8Form form = fp8_form(a.E, a.M, a.K, a.N, f32);
  // (at most: full tiles, and one that is not full for each expert)
  const int64_t tiles_of_rows = a.N / form.rows + std::min(a.E, a.N);
  if (form.m == TILE_M) {
    const int64_t most = tiles_of_rows * ((a.M + TILE_M - 1) / TILE_M);
    auto tiles = [&](auto kernel) {
      return enqueue(kernel, (int)std::min<int64_t>(512, (most + N_XCD - 1) / N_XCD * N_XCD), 256, s, a);
    };
    if (f32) return form.rows == 96 ? tiles(k_fp8_tiles<true, 96, 1>) : tiles(k_fp8_tiles<true, 64, 2>);
    return form.rows == 128 ? tiles(k_fp8_tiles<false, 128, 1>) : tiles(k_fp8_tiles<false, 96, 2>);
  }
  auto split = [&](auto r_c, auto ns_c) {
    constexpr int R = decltype(r_c)::value, NS = decltype(ns_c)::value;
    const int64_t items = tiles_of_rows * ((a.M + 63) / 64) * (4 / R);
    const int grid = (int)std::min<int64_t>(items, R == 4 ? 512 : 1024);
    return enqueue(f32 ? k_fp8_split<true, R, NS> : k_fp8_split<false, R, NS>, grid, 256, s, a);
  };
  using one = std::integral_constant<int, 1>;
  using two = std::integral_constant<int, 2>;
  using four = std::integral_constant<int, 4>;
  if (form.rows == 32) return form.m == 64 ? split(four(), two()) : split(two(), two());
  return form.m == 32 ? split(two(), one()) : split(one(), one());
}

// A thread writes 16 codes: of a row's neighbouring columns, or (TRANS) of 16 rows.
template <bool TRANS>
__global__ __launch_bounds__(256) void k_fp8_pack(const uint8_t *w, int M, int K, int64_t chunks,
                                                  uint8_t *packed) {
  const int G = (K + 127) >> 7, MB64 = (M + 63) >> 6;
  for (int64_t c = blockIdx.x * 256ll + threadIdx.x; c < chunks; c += gridDim.x * 256ll) {
    const int lane = (int)(c & 63), h = (int)(c >> 6) & 1, i = (int)(c >> 7) & 3;
    const int64_t t = c >> 9, em = t / G;
    const int g = (int)(t - em * G), mb = (int)(em % MB64);
    const int64_t e = em / MB64;
    const int r = lane & 15, m = mb * 64 + 32 * (i >> 1) + 8 * (r >> 2) + 4 * (i & 1) + (r & 3);
    const int k = g * 128 + 64 * h + 16 * (lane >> 4);
    uint32_t v[4] = {0, 0, 0, 0};
    if (m < M && k < K) {
      if constexpr (TRANS) {
        const uint8_t *from = w + (e * K + k) * M + m;
#pragma unroll
        for (int b = 0; b < 16; ++b) v[b >> 2] |= (uint32_t)from[(int64_t)b * M] << (8 * (b & 3));
      } else {
        const u32x4 x = *(const u32x4 *)(w + (e * M + m) * K + k);
#pragma unroll
        for (int d = 0; d < 4; ++d) v[d] = x[d];
      }
    }
    *(u32x4 *)(packed + c * 16) = u32x4{v[0], v[1], v[2], v[3]};
  }
}

size_t fp8_packed_bytes(int E, int M, int K) {
  return (size_t)E * ((M + 63) / 64) * ((K + 127) / 128) * 8192;
}

hipError_t launch_fp8_pack(const uint8_t *w, int E, int M, int K, int transpose, uint8_t *packed,
                           hipStream_t s) {
  const int64_t chunks = (int64_t)(fp8_packed_bytes(E, M, K) / 16);
  const int grid = (int)std::min<int64_t>((chunks + 255) / 256, 1 << 20);
  return enqueue(transpose ? k_fp8_pack<true> : k_fp8_pack<false>, grid, 256, s, w, M, K, chunks, packed);
}
