// moe_lora.hip - low-rank adapters of many requests beside shared projections
// (ainfer_moe_lora_apply): y_p += scale_a (x A_a^T) B_a^T, a = the token's adapter.
//
// Batches of requests (an adapter per token: A and B are read for every token, and
// launches and latency count) take dot products in fp32, one token a workgroup:
//   k_lora_dec    a workgroup owns rows of one token's y: a wave per row of A, v to
//                 LDS, then the rows of B, whose loads are in flight before A's.
//                 A is read by every workgroup of the token, which costs less than
//                 a second launch while it is small
//   k_lora_rows   else v = x A^T first, a workgroup per 2 or 4 rows of A
// Prompts (neighbouring tokens share an adapter):
//   k_lora_tile   16 neighbouring tokens are the columns of
//                 v_mfma_f32_16x16x32_bf16, once per distinct adapter among them,
//                 other tokens' columns ignored: no sorting, tokens may name
//                 adapters in any order.  Its products are exact too: bf16 values
//                 enter the MFMA as they are, fp32 values (x, and v) as the sum of three
//                 bf16 (split_bf16).  v never leaves the CU.
// GPU us a call (inside a graph), and the time the bytes of x, y, and each A and B
// used once take at 5.1 TB/s: one token 4096 x 4096 rank 16 4.8 (0.1; a launch alone is
// 2.5), 64 tokens 4096 x (1024 + 1024) rank 16 6.1 (2.2), 16 tokens 5120 x 17408 rank
// 64 14.8 (8.3), 1003 tokens of 7 requests 1024 x 4096 rank 8 in fp32 12.1 (7.3), 4096
// tokens 4096 x 4096 of 24 requests rank 32 29 (19.3), rank 64 45 (21.5), of one
// request rank 32 21 (19.7), 1024 tokens of 16 requests rank 128 34 (10).
//
// What bounds it: batches, the two dependent sweeps over A and B (an HBM latency each)
// and the bytes of B.  Prompts, y's and x's bytes while a tile has one adapter; a tile
// that lies across two requests is two workgroups, and the second shares its CU with
// another tile's: it ends 5 us (rank 16) to 10 (rank 64) after the others.  From 33 ranks
// on, A and B: every tile of 16 tokens takes its adapter's whole rows through L2 and LDS
// (2 MB at rank 128, 1.3 M reads of 128 bytes a call of 1024 tokens) for one column block
// of the MFMAs.
#include "moe_common.h"
#include "moe_internal.h"

namespace {

constexpr int N_CU = 256;
constexpr int TT = 16;       // tokens of an MFMA tile
constexpr int R_WAVES = 4;   // waves of a workgroup: k_lora_rows
constexpr int dec_waves(bool fused) { return fused ? 8 : 4; }  // k_lora_dec

struct LoraArgs {
  const void *x;
  const int32_t *ids, *ranks;
  const float *scales;
  const uint16_t *a[AINFER_LORA_MAX_PROJ], *b[AINFER_LORA_MAX_PROJ];
  void *y[AINFER_LORA_MAX_PROJ];
  int64_t y_ld[AINFER_LORA_MAX_PROJ], x_ld;
  int m[AINFER_LORA_MAX_PROJ];
  float *v;       // [P][T][R], x A^T of a first launch
  int N, R, K, P, T;
  int units;      // groups of 64 rows of y per wave
};

__device__ __forceinline__ int rank_of(const LoraArgs &a, int ad) {
  return a.ranks ? min(max(a.ranks[ad], 0), a.R) : a.R;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

// ---- batches of requests ------------------------------------------------------

__device__ __forceinline__ float wave_sum_f32(float v) {
  auto dpp = [](float x, auto ctrl, auto rows) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value,
                                                      decltype(rows)::value, 0xF, false));
  };
  using std::integral_constant;
  v += dpp(v, integral_constant<int, 0xB1>(), integral_constant<int, 0xF>());
  v += dpp(v, integral_constant<int, 0x4E>(), integral_constant<int, 0xF>());
  v += dpp(v, integral_constant<int, 0x141>(), integral_constant<int, 0xF>());
  v += dpp(v, integral_constant<int, 0x140>(), integral_constant<int, 0xF>());
  v += dpp(v, integral_constant<int, 0x142>(), integral_constant<int, 0xA>());
  v += dpp(v, integral_constant<int, 0x143>(), integral_constant<int, 0xC>());
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// 8 values of x from k
template <bool XF32>
struct X8 {
  u32x4 v[XF32 ? 2 : 1];
  __device__ __forceinline__ void load(const char *row, int k) {
#pragma unroll
    for (int i = 0; i < (XF32 ? 2 : 1); ++i)
      v[i] = *(const u32x4 *)(row + (size_t)k * (XF32 ? 4 : 2) + 16 * i);
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (XF32) return __uint_as_float(v[i / 4][i & 3]);
    return i & 1 ? bf16_hi(v[0][i / 2]) : bf16_lo(v[0][i / 2]);
  }
};
template <bool XF32>
__device__ __forceinline__ void dot8(const X8<XF32> &x, const u32x4 &w, float &acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = fmaf(x.at(2 * i), bf16_lo(w[i]), acc);
    acc = fmaf(x.at(2 * i + 1), bf16_hi(w[i]), acc);
  }
}

// x . A's NR rows, step apart, over the k of wave `wave` of W (runs of 512 in
// turn), four runs' loads in flight; every lane gets the sums
template <bool XF32, int NR, int W>
__device__ __forceinline__ void row_dots(const char *xr, const uint16_t *ar, size_t step, int K,
                                         int wave, int lane, float (&sum)[NR]) {
  constexpr int U = 4, RUN = 512 * W;
  float acc[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r) acc[r][0] = acc[r][1] = 0.0f;
  const int k1 = wave * 512 + lane * 8;
  auto runs = [&](int k0, auto whole) {  // runs k0, k0 + RUN, ...
    X8<XF32> x[U];
    u32x4 w[U][NR];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + k1 + RUN * u;
      if constexpr (!decltype(whole)::value) {
#pragma unroll
        for (auto &v : x[u].v) v = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < NR; ++r) w[u][r] = (u32x4){0, 0, 0, 0};
        if (k >= K) continue;  // K is a multiple of 8
      }
      x[u].load(xr, k);
#pragma unroll
      for (int r = 0; r < NR; ++r) w[u][r] = *(const u32x4 *)(ar + r * step + k);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < NR; ++r) dot8(x[u], w[u][r], acc[r][u & 1]);
  };
  int k0 = 0;
  for (; k0 + U * RUN <= K; k0 += U * RUN) runs(k0, std::true_type());
  if (k0 < K) runs(k0, std::false_type());
#pragma unroll
  for (int r = 0; r < NR; ++r) sum[r] = wave_sum_f32(acc[r][0] + acc[r][1]);
}

// v of one token: rows first, first + step, ... below rank, two at a time
template <bool XF32, typename Put>
__device__ __forceinline__ void token_rows(const LoraArgs &a, int p, int t, int ad, int first,
                                           int step, int rank, int lane, Put put) {
  const char *xr = (const char *)a.x + (size_t)t * a.x_ld * (XF32 ? 4 : 2);
  const uint16_t *A = a.a[p] + (size_t)ad * a.R * a.K;
  int r = first;
  for (; r + step < rank; r += 2 * step) {
    float s[2];
    row_dots<XF32, 2, 1>(xr, A + (size_t)r * a.K, (size_t)step * a.K, a.K, 0, lane, s);
    put(r, s[0]);
    put(r + step, s[1]);
  }
  if (r < rank) {
    float s[1];
    row_dots<XF32, 1, 1>(xr, A + (size_t)r * a.K, 0, a.K, 0, lane, s);
    put(r, s[0]);
  }
}

// NR rows of A a workgroup, its waves 512 k after each other: all of a row's loads
// are in flight up to K = 8192
template <int NR, bool XF32>
__global__ __launch_bounds__(64 * R_WAVES) void k_lora_rows(LoraArgs a) {
  __shared__ float s_sum[R_WAVES][NR];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x, p = blockIdx.z, r0 = blockIdx.y * NR;
  const int ad = a.ids[t];
  if (ad < 0 || ad >= a.N) return;
  const int rank = rank_of(a, ad);
  if (r0 >= rank) return;
  const char *xr = (const char *)a.x + (size_t)t * a.x_ld * (XF32 ? 4 : 2);
  const uint16_t *A = a.a[p] + ((size_t)ad * a.R + r0) * a.K;  // R is a multiple of NR
  float sum[NR];
  row_dots<XF32, NR, R_WAVES>(xr, A, a.K, a.K, wave, lane, sum);
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < NR; ++r) s_sum[wave][r] = sum[r];
  }
  __syncthreads();
  if (wave == 0 && lane < NR) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < R_WAVES; ++w) v += s_sum[w][lane];
    a.v[((size_t)p * a.T + t) * a.R + r0 + lane] = v;
  }
}

template <int M>
__device__ __forceinline__ float xor_lane(float v) {
  if constexpr (M == 1)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false));
  else if constexpr (M == 2)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false));
  else
    return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), (M << 10) | 0x1F));
}
// Lane s of a run of LR lanes gets the run's sum of d[s]: at each step a lane
// keeps one half of its values and receives its partner's of the same half.
template <int LR, int M = LR / 2>
__device__ __forceinline__ void sum_transpose(float (&d)[LR], int s) {
  if constexpr (M >= 1) {
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const bool up = s & M;
      const float keep = up ? d[j + M] : d[j], send = up ? d[j] : d[j + M];
      d[j] = keep + xor_lane<M>(send);
    }
    sum_transpose<LR, M / 2>(d, s);
  }
}

// One token's rows of y.  LR lanes share a row of B, 8 of its columns each, so a
// wave reads 1 KB of consecutive rows per load; LR loads cover 64 rows, whose
// sums end one per lane, in order.  FUSED: v is computed here, in LDS, with the
// first rows of B and y already in flight.
template <int LR, bool FUSED, bool XF32, bool YF32>
__global__ __launch_bounds__(64 * dec_waves(FUSED)) void k_lora_dec(LoraArgs a) {
  constexpr int D_WAVES = dec_waves(FUSED);
  constexpr int G = LR >= 8 ? 1 : 8 / LR;  // groups of 64 rows in flight
  constexpr int RW = 64 / LR;              // rows of a load
  __shared__ float s_v[FUSED ? 128 : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x, p = blockIdx.z, M = a.m[p];
  const int ad = a.ids[t];
  if (ad < 0 || ad >= a.N) return;
  const int rank = rank_of(a, ad);
  if (rank == 0) return;
  const int g0 = (blockIdx.y * D_WAVES + wave) * a.units;  // this wave's groups of 64 rows
  const int g1 = min(g0 + a.units, (M + 63) / 64);
  if (blockIdx.y * D_WAVES * a.units * 64 >= M) return;
  const float scale = a.scales ? a.scales[ad] : 1.0f;
  const int s = lane & (LR - 1), rs = lane / LR, r0 = s * 8;
  const uint16_t *B = a.b[p] + (size_t)ad * M * a.R;
  const size_t yrow = (size_t)t * a.y_ld[p];

  u32x4 w[G][LR];
  float y[G];
  auto load = [&](int g) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      if (g + i >= g1) continue;
#pragma unroll
      for (int j = 0; j < LR; ++j) {
        w[i][j] = (u32x4){0, 0, 0, 0};
        const int m = min((g + i) * 64 + j * RW + rs, M - 1);
        if (r0 < rank) w[i][j] = *(const u32x4 *)(B + (size_t)m * a.R + r0);
      }
      const int m = (g + i) * 64 + s * RW + rs;
      if (m < M)
        y[i] = YF32 ? ((const float *)a.y[p])[yrow + m]
                    : bf16_to_f32(((const uint16_t *)a.y[p])[yrow + m]);
    }
  };
  load(g0);
  __builtin_amdgcn_sched_barrier(0);
  float v[8];
  if constexpr (FUSED) {
    token_rows<XF32>(a, p, t, ad, wave, D_WAVES, rank, lane, [&](int r, float d) {
      if (lane == 0) s_v[r] = d;
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r0 + i < rank ? s_v[r0 + i] * scale : 0.0f;
  } else {
    const float *src = a.v + ((size_t)p * a.T + t) * a.R;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r0 + i < rank ? src[r0 + i] * scale : 0.0f;
  }
  u32x4 keep;  // clears B's columns from rank on (they may hold anything)
#pragma unroll
  for (int i = 0; i < 4; ++i)
    keep[i] = (r0 + 2 * i < rank ? 0xFFFFu : 0u) | (r0 + 2 * i + 1 < rank ? 0xFFFF0000u : 0u);
  for (int g = g0; g < g1; g += G) {
    if (g != g0) load(g);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      if (g + i >= g1) continue;
      float d[LR];
#pragma unroll
      for (int j = 0; j < LR; ++j) {
        const u32x4 b = w[i][j] & keep;
        float acc = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc = fmaf(v[2 * e], bf16_lo(b[e]), acc);
          acc = fmaf(v[2 * e + 1], bf16_hi(b[e]), acc);
        }
        d[j] = acc;
      }
      sum_transpose<LR>(d, s);
      const int m = (g + i) * 64 + s * RW + rs;
      if (m < M) {
        if constexpr (YF32)
          ((float *)a.y[p])[yrow + m] = y[i] + d[0];
        else
          ((uint16_t *)a.y[p])[yrow + m] = f32_to_bf16(y[i] + d[0]);
      }
    }
  }
}

// ---- prompts ------------------------------------------------------------------

// NS values that sum to x, each exact in bf16 (x's 24 bits from the top, 8 at a
// time), as fp32 with the low half clear.  inf and NaN stay in the first.
constexpr int NS = 3;
__device__ __forceinline__ void split_bf16(float x, float (&s)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    s[i] = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    x = x == s[i] ? 0.0f : x - s[i];
  }
}
// the high halves of two such values
__device__ __forceinline__ uint32_t pack_hi(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// a lane's 4 values of one token's y: neighbours (VEC), or 16 apart, one access each
template <bool YF32, bool VEC>
struct YRun {
  uint32_t v[YF32 || !VEC ? 4 : 2];
  // at: of value j
  template <class At>
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, At at_j) {
    const uint32_t at = at_j(0);
    if constexpr (!VEC) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = YF32 ? __builtin_amdgcn_raw_buffer_load_b32(r, at_j(j), 0, 0)
                    : __builtin_amdgcn_raw_buffer_load_b16(r, at_j(j), 0, 0);
    } else if constexpr (YF32) {
      const u32x4 t = buf_load16(r, at);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = t[j];
    } else {
      const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
      v[0] = t[0];
      v[1] = t[1];
    }
  }
  // += d, rounded once
  __device__ __forceinline__ void add(const YRun &y, float d0, float d1, float d2, float d3) {
    const float d[4] = {d0, d1, d2, d3};
    if constexpr (YF32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(__uint_as_float(y.v[j]) + d[j]);
    } else if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        v[j] = bf16x2_bits(bf16_lo(y.v[j]) + d[2 * j], bf16_hi(y.v[j]) + d[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = f32_to_bf16(bf16_lo(y.v[j]) + d[j]);
    }
  }
  template <class At>
  __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, At at_j) const {
    const uint32_t at = at_j(0);
    if constexpr (!VEC) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (YF32) __builtin_amdgcn_raw_buffer_store_b32(v[j], r, at_j(j), 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)v[j], r, at_j(j), 0, 0);
      }
    } else if constexpr (YF32)
      __builtin_amdgcn_raw_buffer_store_b128((u32x4){v[0], v[1], v[2], v[3]}, r, at, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b64((u32x2){v[0], v[1]}, r, at, 0, 0);
  }
};

// ids of a tile's tokens, one per lane below 16; -1 = none
__device__ __forceinline__ int tile_ids(const LoraArgs &a, int t0, int lane) {
  int id = -1;
  if (lane < TT && t0 + lane < a.T) id = a.ids[t0 + lane];
  return id >= 0 && id < a.N ? id : -1;
}

__device__ __forceinline__ void lds_order() {  // a wave's own LDS writes before its reads
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// 16 rows of CK columns, read by one wave as whole rows (LPR lanes a row, 16
// bytes each) and handed to the MFMA's layout (lane (q, col): row col, columns
// 32 s + 8 q) through 16 x CK x 2 bytes of its LDS.  A load straight into that
// layout touches a line per lane, four times what whole rows do.  Piece c of
// row r lies at place c ^ swz(r) of its row, so that neither side meets a bank
// twice.
template <int CK>
struct Panel {
  static constexpr int LPR = CK / 8, LOADS = LPR / 4, RPL = 64 / LPR;
  static __device__ __forceinline__ int swz(int row) { return CK == 128 ? row & 15 : (row >> 1) & 7; }
  u32x4 v[LOADS];
  // rows row0 + i * RPL + lane / LPR, columns k0 + (lane % LPR) * 8 of a matrix of
  // rows of K columns (at most 16 MB); 0 past its last row and column
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t m, int row0, int k0, int K, int lane) {
    const int k = k0 + (lane & (LPR - 1)) * 8;
    const uint32_t at = k < K ? (uint32_t)(lane / LPR * K + k) * 2 : BUF_OOB;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      v[i] = buf_load16(m, at + (uint32_t)((row0 + i * RPL) * K) * 2);
  }
  __device__ __forceinline__ void to_lds(u32x4 *buf, int lane) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int r = i * RPL + lane / LPR;
      buf[r * LPR + ((lane & (LPR - 1)) ^ swz(r))] = v[i];
    }
  }
  static __device__ __forceinline__ void frags(const u32x4 *buf, int lane, u32x4 (&f)[CK / 32]) {
    const int col = lane & 15, q = lane >> 4;
#pragma unroll
    for (int s = 0; s < CK / 32; ++s) f[s] = buf[col * LPR + ((s * 4 + q) ^ swz(col))];
  }
};

// the same of fp32 rows: the wave splits what it read, one plane of bf16 each
struct PanelF32 {
  static constexpr int CK = 64;
  u32x4 v[4];  // row i * 4 + lane / 16, columns k0 + (lane % 16) * 4
  __device__ __forceinline__ void to_lds(u32x4 *buf, int lane) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 4 + lane / 16, piece = (lane & 15) >> 1;
      float e[4][NS];
#pragma unroll
      for (int j = 0; j < 4; ++j) split_bf16(__uint_as_float(v[i][j]), e[j]);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        u32x2 w = {pack_hi(e[0][s], e[1][s]), pack_hi(e[2][s], e[3][s])};
        u32x4 *row = buf + s * 128 + r * 8;
        ((u32x2 *)(row + (piece ^ Panel<CK>::swz(r))))[lane & 1] = w;
      }
    }
  }
};

// One adapter's tokens of a tile of 16, all of K, then all of this workgroup's
// rows of y.  blockIdx.x: tile, blockIdx.y: projection and part of its rows,
// blockIdx.z: which distinct adapter of the tile (slowest, so that the first adapters
// of all tiles and parts start first, on CUs of their own; a workgroup of an adapter
// that a tile lacks ends after one load).
//   1. v = A x^T: a wave takes every T_WAVES-th chunk of CK columns; A's next rows
//      are read while the last ones are multiplied.  The sums meet in LDS.
//   2. v scaled, split and laid out for the MFMA.
//   3. units of 64 rows of B: column c of MFMA j is row 4 c + j, so that a lane
//      ends with 4 consecutive values of y of each of its 4 tokens (VEC: y in
//      whole pieces of 4; else row 16 j + c, so that 16 lanes reach a line
//      together).  B's rows are read whole and turned in LDS as A's; what the
//      next unit reads of B and y is in flight meanwhile.
// STAGES V: 1 alone, of 32 rows of A (blockIdx.y: projection and which), v
// to memory; Y: 2 and 3 of that v.
enum { STAGES_VY, STAGES_V, STAGES_Y };
constexpr int tile_waves(int stages) { return stages == STAGES_Y ? 4 : 8; }
// Two workgroups a CU (128 registers) where they fit: a tile with a second adapter
// then need not wait for a first round.  4096 tokens of 24 requests, 4096 x 4096, rank
// 64 44.4 us (46 with one), 8192 tokens of 30 79 (88).  Ranks 49 to 64 with y in single
// values fit only with v's parts read from LDS for every product: 4096 x 4097 50 to 56
// (55 to 57 with one), 2048 tokens of 12, 2048 x 2049, rank 56 22.5 (18.3).
constexpr bool tile_two(int lp, bool yf32, bool vec) {
  return lp <= 6 || (lp == 8 && !yf32 && vec);
}
// waves a SIMD holds: of STAGES_Y the LDS allows three workgroups, from 65 ranks two
constexpr int tile_occupancy(int stages, int lp, bool yf32, bool vec) {
  return stages == STAGES_Y ? (lp <= 8 ? 3 : 2) : tile_two(lp, yf32, vec) ? 4 : 2;
}
template <int STAGES, int LP, bool XF32, bool YF32, bool VEC>
__global__ __launch_bounds__(64 * tile_waves(STAGES),
                             tile_occupancy(STAGES, LP, YF32, VEC)) void k_lora_tile(LoraArgs a) {
  constexpr int T_WAVES = tile_waves(STAGES);
  // blocks of 16 rows of A (4 also for 33 to 48 rows: two panels in flight divide them)
  constexpr int NRB = LP <= 2 ? 1 : LP == 6 ? 4 : LP / 2;
  constexpr int NRK = (NRB + 1) / 2;
  constexpr int CK = XF32 ? 64 : 128, KS = CK / 32, NX = XF32 ? NS : 1;
  // panels of A in flight; a block's place among them is the same in every chunk
  constexpr int RING = NRB < 3 ? NRB : tile_two(LP, YF32, VEC) ? 2 : NRB % 4 ? 3 : 4;
  static_assert(NRB % RING == 0, "");
  constexpr int STAGE = NRK <= 2 ? 512 : NRK * 256;  // 16-byte pieces of a wave's LDS
  constexpr int XPART = XF32 ? 384 : 256;  // the x panel's share of it
  __shared__ u32x4 s_stage[T_WAVES][STAGE + 64];
  __shared__ u32x2 s_v[NRK][NS][64][2];
  const int lane0 = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbouring tiles on one XCD, whose L2 then holds their adapters
  const int t0 = xcd_remap(blockIdx.x, gridDim.x) * TT;
  const int p = blockIdx.y % a.P, part = blockIdx.y / a.P;
  const int M = a.m[p];
  const int id = tile_ids(a, t0, lane0);
  const int row0 = STAGES == STAGES_V ? part * NRB * 16 : 0;  // of A
  uint32_t rem = (uint32_t)__ballot(id >= 0);  // 16 tokens
  const int u0 = part * a.units * T_WAVES, u_end = min(u0 + a.units * T_WAVES, (M + 63) / 64);
  if (STAGES != STAGES_V && u0 >= u_end) return;
  for (int nth = 0; rem; ++nth) {
    const int ad = __builtin_amdgcn_readlane(id, __builtin_ctz(rem));
    const uint32_t mask = (uint32_t)__ballot(id == ad) & rem;
    rem &= ~mask;
    if (nth % (int)gridDim.z != (int)blockIdx.z) continue;
    const int rank = rank_of(a, ad);
    if (rank <= row0) continue;
    const float scale = a.scales ? a.scales[ad] : 1.0f;
    // opaque, so that what depends on the lane is computed again for each adapter
    // and not held in registers across this loop
    const int lane = tid_opaque() & 63;
    u32x4 *stage = s_stage[wave];

    // 1.
    f32x4 acc[NRB];
#pragma unroll
    for (int r = 0; r < NRB; ++r) acc[r] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if constexpr (STAGES != STAGES_Y) {
      const __amdgpu_buffer_rsrc_t A =
          make_rsrc(a.a[p] + (size_t)ad * a.R * a.K, (uint32_t)(a.R * a.K) * 2);
      const int nc = (a.K + CK - 1) / CK;
      Panel<CK> pa[RING];
      using XPanel = typename std::conditional<XF32, PanelF32, Panel<CK>>::type;
      XPanel px;
      auto load_a = [&](int r, int c) { pa[r % RING].load(A, row0 + r * 16, c * CK, a.K, lane); };
      // the tile's rows of x; rows past the last token are never multiplied into a
      // token's column, and read as 0
      const int xsz = XF32 ? 4 : 2;
      const __amdgpu_buffer_rsrc_t X =
          make_rsrc((const char *)a.x + (size_t)t0 * a.x_ld * xsz, 0x7FFFFFFFu);
      const uint32_t xpitch = (uint32_t)a.x_ld * xsz;
      uint32_t x_row[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 4 + lane / 16;
        x_row[i] = t0 + r < a.T ? r * xpitch : BUF_OOB;
      }
      auto load_x = [&](int c) {
        const int k = c * CK + (lane & 15) * (16 / xsz);  // 16 lanes a row
#pragma unroll
        for (int i = 0; i < 4; ++i) px.v[i] = buf_load16(X, k < a.K ? x_row[i] + k * xsz : BUF_OOB);
      };
      // chunks from nc on read as 0, without a branch: a branch around a load or a
      // store makes every later wait a wait for all of them
      load_x(wave);
#pragma unroll
      for (int r = 0; r < RING; ++r) load_a(r, wave);
      for (int c = wave; c < nc; c += T_WAVES) {
        const int next = c + T_WAVES;
        u32x4 xf[NX][KS];
        px.to_lds(stage, lane);
        load_x(next);
        lds_order();
#pragma unroll
        for (int s = 0; s < NX; ++s) Panel<CK>::frags(stage + s * 128, lane, xf[s]);
#pragma unroll
        for (int r = 0; r < NRB; ++r) {
          u32x4 *buf = stage + XPART;
          pa[r % RING].to_lds(buf, lane);
          if (r + RING < NRB) load_a(r + RING, c);
          else load_a((r + RING) % NRB, next);
          lds_order();
          u32x4 af[KS];
          Panel<CK>::frags(buf, lane, af);
#pragma unroll
          for (int s = 0; s < NX; ++s)
#pragma unroll
            for (int k = 0; k < KS; ++k) acc[r] = mfma_bf16_16x16x32(af[k], xf[s][k], acc[r]);
          lds_order();
        }
      }
    }
    const int lane_y = tid_opaque() & 63, col_y = lane_y & 15, q_y = lane_y >> 4;
    // the sums of the waves: ranks row0 + rb * 16 + q_y * 4 .. + 3 of token col
    auto to_red = [&]() {
      f32x4 *red = (f32x4 *)s_stage;  // [T_WAVES][NRB][64]
#pragma unroll
      for (int r = 0; r < NRB; ++r) red[(wave * NRB + r) * 64 + lane_y] = acc[r];
    };
    auto from_red = [&](int rb) {
      const f32x4 *red = (const f32x4 *)s_stage;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < T_WAVES; ++w) v += red[(w * NRB + rb) * 64 + lane_y];
      return v;
    };
    float *const v_tok = a.v + ((size_t)p * a.T + t0 + col_y) * a.R;  // of token col
    if constexpr (STAGES == STAGES_V) {
      __syncthreads();  // every wave is done with its stage
      to_red();
      __syncthreads();
      for (int rb = wave; rb < NRB; rb += T_WAVES) {
        const f32x4 v = from_red(rb);
        const int r0 = row0 + rb * 16 + q_y * 4;
        if ((mask >> col_y) & 1 && r0 < a.R) *(f32x4 *)(v_tok + r0) = v;
      }
    } else {
      const uint32_t own = mask >> (q_y * 4);  // bit i: this lane's token q * 4 + i
      constexpr int CP = NRK * 4;              // pieces of a row of B, padded
      const int cpr = a.R / 8;
      const __amdgpu_buffer_rsrc_t B =
          make_rsrc(a.b[p] + (size_t)ad * M * a.R, (uint32_t)M * a.R * 2);
      u32x4 w[LP];
      YRun<YF32, VEC> y[4];
      const int ysz = YF32 ? 4 : 2;
      const __amdgpu_buffer_rsrc_t Y =
          make_rsrc((const char *)a.y[p] + (size_t)t0 * a.y_ld[p] * ysz, 0x7FFFFFFFu);
      const uint32_t ypitch = (uint32_t)a.y_ld[p] * ysz;
      uint32_t y_tok[4];  // this lane's tokens q * 4 + i, or past the buffer
#pragma unroll
      for (int i = 0; i < 4; ++i) y_tok[i] = (own >> i) & 1 ? (q_y * 4 + i) * ypitch : BUF_OOB;
      auto y_at = [&](int u, int i, int j) {
        const int m = u * 64 + (VEC ? 4 * col_y + j : 16 * j + col_y);
        return m < M ? y_tok[i] + m * ysz : BUF_OOB;
      };
      auto load_b = [&](int u) {
#pragma unroll
        for (int i = 0; i < LP; ++i)  // piece i * 64 + lane of the unit
          w[i] = buf_load16(B, (uint32_t)(u * cpr + i) * 1024 + lane_y * 16);
      };
      auto load_y = [&](int u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i].load(Y, [&](int j) { return y_at(u, i, j); });
      };
      int u = u0 + wave;
      load_b(u);
      load_y(u);
      if constexpr (STAGES == STAGES_VY) {
        __syncthreads();  // every wave is done with its stage
        to_red();
        __syncthreads();
      }
      // 2.
      for (int rb = wave; rb < 2 * NRK; rb += T_WAVES) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        float e[4][NS];
        const int r0 = rb * 16 + q_y * 4;
        if constexpr (STAGES == STAGES_VY) {
          if (rb < NRB) v = from_red(rb);
        } else {
          // another adapter's tokens of the tile are never multiplied into this one's
          if ((mask >> col_y) & 1 && r0 < rank) v = *(const f32x4 *)(v_tok + r0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) split_bf16(r0 + i < rank ? v[i] * scale : 0.0f, e[i]);
        const int slot = ((r0 & 31) >> 3) * 16 + col_y;
#pragma unroll
        for (int s = 0; s < NS; ++s)
          s_v[rb >> 1][s][slot][(r0 >> 2) & 1] =
              (u32x2){pack_hi(e[0][s], e[1][s]), pack_hi(e[2][s], e[3][s])};
      }
      __syncthreads();

      // 3.
      // piece i * 64 + lane of a unit: its place in the stage.  4 rows (a column of
      // the MFMAs) are 4 CP pieces, turned by the column so that neither side meets a
      // bank twice.
      int place[LP];
#pragma unroll
      for (int i = 0; i < LP; ++i) {
        const int l = i * 64 + lane_y, row = l / cpr, ch = l - row * cpr;
        const int c = VEC ? row >> 2 : row & 15, j = VEC ? row & 3 : row >> 4;
        place[i] = row < 64 ? c * 4 * CP + ((j * CP + ch) ^ c) : STAGE + lane_y;
      }
      u32x4 keep;  // clears B's columns from rank on (they may hold anything) in rank's block of 32
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = q_y * 8 + 2 * i, n = rank & 31;
        keep[i] = (r < n ? 0xFFFFu : 0u) | (r + 1 < n ? 0xFFFF0000u : 0u);
      }
      u32x4 vf[NRK][NS];
#pragma unroll
      for (int rb = 0; rb < NRK; ++rb)
#pragma unroll
        for (int s = 0; s < NS; ++s) vf[rb][s] = *(const u32x4 *)s_v[rb][s][lane_y];

      // d = v B^T of unit u, and the next unit's rows on their way
      auto product = [&](int u, f32x4 (&d)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < LP; ++i) stage[place[i]] = w[i];
        load_b(u + T_WAVES);
        lds_order();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int rb = 0; rb < NRK; ++rb) {
            u32x4 b = stage[col_y * 4 * CP + ((j * CP + rb * 4 + q_y) ^ col_y)];
            // from rank on B may hold anything: its block of 32 is masked, later ones are left out
            if (rb * 32 + 32 > rank) b = rb * 32 < rank ? b & keep : (u32x4){0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) d[j] = mfma_bf16_16x16x32(vf[rb][s], b, d[j]);
          }
        lds_order();
      };
      for (; u < u_end; u += T_WAVES) {
        f32x4 d[4];
        product(u, d);
        YRun<YF32, VEC> o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i].add(y[i], d[0][i], d[1][i], d[2][i], d[3][i]);
        load_y(u + T_WAVES);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i].store(Y, [&](int j) { return y_at(u, i, j); });
      }
    }
    if (rem) __syncthreads();  // the stage is the next adapter's
  }
}

// ---- launches -----------------------------------------------------------------

int div_up(int a, int b) { return (a + b - 1) / b; }

// Up to this many tokens a call is taken as a batch of requests.  GPU us by tokens and
// by tiles: every token another of 64 adapters, 256 tokens 4096 x 4096 rank 16 14.6 and
// 32, 1024 x 4096 rank 8 fp32 7.8 and 25.5, 2048 x (2048 + 2048) rank 64 35 and 51;
// prompts of 4 requests, 128 tokens rank 16 8.3 and 7.2, 256 9.9 and 7.6, rank 8 5.8 and
// 7.1, rank 64 20 and 14; of 16 requests 256 tokens 11.2 and 11.3, 6.4 and 9.4, 22 and 16.
constexpr int DEC_MAX_T = 256;

// v in every workgroup of a token, or by k_lora_rows first.  us, K 4096, M 4096
// (8 workgroups a token up to 64 tokens, 4 and 2 at 128 and 256), fused and not:
// rank 16, T 1 4.8 and 6.3, 64 8.5 and 9.1, 128 10.3 and 13.4, 256 14.7 and 17.4;
// rank 32, T 1 6.5 and 6.5, 16 6.8 and 6.2, 64 13.3 and 11.3; rank 64, T 1 9.9 and
// 6.3.  K 5120, M 17408, rank 16, T 16 (17 workgroups a token): 9.7 and 8.3.
constexpr size_t FUSED_BYTES = 256 << 10;  // of an adapter's A
constexpr size_t FUSED_AGAIN = 64 << 20;   // of A read again by a token's further workgroups
bool fuse(size_t bytes_a, int tokens, int workgroups) {
  const size_t again = (size_t)(workgroups - 1) * tokens * bytes_a;
  return bytes_a <= FUSED_BYTES && again * (workgroups > 8 ? 2 : 1) <= FUSED_AGAIN;
}
// Workgroups of k_lora_dec: fused, two on each CU, all at once, as each reads A (T 192
// rank 16, 4096 x 4096, 3 and 2 a token: 15.6 and 12.8 us); alone, about this many waves,
// for the loads in flight (rank 32, T 256 27.3 at 4096, 23.8 at 8192, 25.5 at 16384)
constexpr int DEC_WAVES_WANTED = 8192;
// k_lora_rows: two rows a workgroup, four from this many rows in the call (fewer
// workgroups for equal time: rank 128, T 256 76.9 and 77.3 us)
constexpr int ROWS_TWO = 4096;
// k_lora_tile in two launches where further parts of y's rows would read more of A
// again, us in one and in two: T 300, 4096 x 4096, rank 64 (70 MB) 23.9 and 15.1, T 512,
// rank 96 (176 MB) 33.2 and 21.7, T 1024, rank 128 (201 MB) 52.9 and 36.5, T 934, 704 x
// 685 x 2, rank 112 (19 MB) 30.9 and 27.3, T 300, 1024 x 1024, rank 40 (11 MB) 7.2 and
// 8.6; of tiles that fill the card, T 2048, 4096 x 1024 x 2, rank 48 (0) 25.4 and 30.4.
constexpr size_t TILE_AGAIN = 16 << 20;

template <int LR, bool FUSED>
void launch_dec(const LoraArgs &a, dim3 grid, bool xf32, bool yf32, hipStream_t s) {
  const dim3 b(64 * dec_waves(FUSED));
  if constexpr (FUSED) {
    if (xf32) {
      if (yf32) k_lora_dec<LR, true, true, true><<<grid, b, 0, s>>>(a);
      else k_lora_dec<LR, true, true, false><<<grid, b, 0, s>>>(a);
      return;
    }
  }
  if (yf32) k_lora_dec<LR, FUSED, false, true><<<grid, b, 0, s>>>(a);
  else k_lora_dec<LR, FUSED, false, false><<<grid, b, 0, s>>>(a);
}
template <bool FUSED>
void launch_dec_lr(const LoraArgs &a, dim3 grid, bool xf32, bool yf32, hipStream_t s) {
  if (a.R <= 8) launch_dec<1, FUSED>(a, grid, xf32, yf32, s);
  else if (a.R <= 16) launch_dec<2, FUSED>(a, grid, xf32, yf32, s);
  else if (a.R <= 32) launch_dec<4, FUSED>(a, grid, xf32, yf32, s);
  else if (a.R <= 64) launch_dec<8, FUSED>(a, grid, xf32, yf32, s);
  else launch_dec<16, FUSED>(a, grid, xf32, yf32, s);
}
template <int STAGES, int LP, bool XF32>
void launch_tile(const LoraArgs &a, dim3 grid, bool yf32, bool vec, hipStream_t s) {
  const dim3 b(64 * tile_waves(STAGES));
  if (yf32) {
    if (vec) k_lora_tile<STAGES, LP, XF32, true, true><<<grid, b, 0, s>>>(a);
    else k_lora_tile<STAGES, LP, XF32, true, false><<<grid, b, 0, s>>>(a);
  } else {
    if (vec) k_lora_tile<STAGES, LP, XF32, false, true><<<grid, b, 0, s>>>(a);
    else k_lora_tile<STAGES, LP, XF32, false, false><<<grid, b, 0, s>>>(a);
  }
}
template <int LP>
void launch_tile_vy(const LoraArgs &a, dim3 grid, bool xf32, bool yf32, bool vec, hipStream_t s) {
  if (xf32) launch_tile<STAGES_VY, LP, true>(a, grid, yf32, vec, s);
  else launch_tile<STAGES_VY, LP, false>(a, grid, yf32, vec, s);
}

}  // namespace

// v of the calls of two launches
size_t lora_workspace_bytes(const ainfer_moe_lora &l, int max_tokens) {
  const size_t n = (size_t)max_tokens * l.n_proj * l.rank * sizeof(float);
  return n > 256 ? (n + 255) & ~(size_t)255 : 256;
}

hipError_t launch_lora(const ainfer_moe_lora &l, const void *x, int64_t x_ld, const int32_t *ids,
                       int T, void *const *y, const int64_t *y_ld, void *ws, hipStream_t s) {
  LoraArgs a;
  a.x = x;
  a.ids = ids;
  a.ranks = l.ranks;
  a.scales = l.scales;
  a.x_ld = x_ld;
  a.v = (float *)ws;
  a.N = l.n_adapters;
  a.R = l.rank;
  a.K = l.in;
  a.P = l.n_proj;
  a.T = T;
  const bool yf32 = l.y_dtype == AINFER_ACT_F32, xf32 = l.x_dtype == AINFER_ACT_F32;
  const int ysz = yf32 ? 4 : 2;
  int m_most = 1;
  bool tiled = T > DEC_MAX_T && (15 * x_ld + l.in) * (xf32 ? 4 : 2) < INT32_MAX;
  bool vec = true;  // every y in whole pieces of 4 values
  for (int p = 0; p < AINFER_LORA_MAX_PROJ; ++p) {
    const bool on = p < l.n_proj;
    a.a[p] = on ? (const uint16_t *)l.a[p] : nullptr;
    a.b[p] = on ? (const uint16_t *)l.b[p] : nullptr;
    a.y[p] = on ? y[p] : nullptr;
    a.y_ld[p] = on ? y_ld[p] : 0;
    a.m[p] = on ? l.out[p] : 0;
    if (on && ((uintptr_t)y[p] % (4 * ysz) || y_ld[p] % 4 || l.out[p] % 4)) vec = false;
    // k_lora_tile's offsets within a tile are 32-bit
    if (on && (15 * y_ld[p] + l.out[p]) * ysz >= INT32_MAX) tiled = false;
    if (on && l.out[p] > m_most) m_most = l.out[p];
  }
  if (!tiled) {
    const int groups = div_up(m_most, 64);
    auto grid = [&](bool fused) {
      const int waves = dec_waves(fused);
      if (fused) {
        const int each = 2 * N_CU / (T * l.n_proj);  // workgroups a token
        a.units = div_up(groups, waves * (each < 1 ? 1 : each));
      } else {
        const int64_t all = (int64_t)groups * T * l.n_proj;  // past 2^31 at pitched large calls
        a.units = (int)((all + DEC_WAVES_WANTED - 1) / DEC_WAVES_WANTED);
      }
      return dim3(T, div_up(groups, a.units * waves), l.n_proj);
    };
    const size_t bytes_a = (size_t)l.rank * l.in * 2;
    dim3 g = grid(true);
    if (fuse(bytes_a, T * l.n_proj, g.y)) {
      launch_dec_lr<true>(a, g, xf32, yf32, s);
    } else {
      g = grid(false);
      const bool four = l.rank * T * l.n_proj > ROWS_TWO;
      const dim3 gr(T, l.rank / (four ? 4 : 2), l.n_proj);
      const dim3 b(64 * R_WAVES);
      if (xf32 && four) k_lora_rows<4, true><<<gr, b, 0, s>>>(a);
      else if (xf32) k_lora_rows<2, true><<<gr, b, 0, s>>>(a);
      else if (four) k_lora_rows<4, false><<<gr, b, 0, s>>>(a);
      else k_lora_rows<2, false><<<gr, b, 0, s>>>(a);
      launch_dec_lr<false>(a, g, xf32, yf32, s);
    }
    return hipGetLastError();
  }
  const int tiles = div_up(T, TT), units = div_up(m_most, 64), cpr = l.rank / 8;
  // a multiple of the XCDs, so that blockIdx.x alone tells the XCD
  const int gx = div_up(tiles, N_XCD) * N_XCD;
  // a.units and how many parts of y's rows, of about `want`
  auto split = [&](int want, int waves) {
    a.units = div_up(units, want * waves);
    return div_up(units, a.units * waves);
  };
  // workgroups of a tile, which share its adapters: as many as two on each CU, and
  // some (with 2 and 4, 4096 x 4096: T 4096, rank 16, 96 requests 34.0 us and 24.9, rank
  // 32, 24 requests 30.4 and 28.2; of a second launch, which has more workgroups of
  // less work, T 512, rank 96 21.8 and 24.7, T 300, rank 64 15.1 and 17.4)
  auto slots = [&](int others, int least) {
    int n = 2 * N_CU / others;
    n = n < least ? least : n > TT ? TT : n;
    return n < l.n_adapters ? n : l.n_adapters;
  };
  // parts of y's rows, each of which computes v again, while tiles leave CUs idle: on
  // half of them (the others are for second adapters of a tile), and fewer where v is
  // most of the work.  us with 1, 2, 4 parts: T 1024, 4096 x 4096, rank 32, 16.6, 13.9,
  // 18.4, T 1003, 1024 x 4096 fp32, rank 8, 14.3, 12.1, 13.2; T 998, 2136 x 1195 of fp32,
  // rank 56, with 1 and 2 17.4 and 22.3; T 1641, 576 x 4239 of fp32, rank 24, 27.7 and 21.3
  const int64_t v_bytes = (int64_t)l.in * (l.rank * 2 + TT * (xf32 ? 4 : 2));
  const int64_t y_bytes = (int64_t)m_most * (l.rank * 2 + TT * 2 * ysz);
  const int idle = N_CU / (tiles * l.n_proj);
  int64_t most = 2 * idle * y_bytes / (5 * v_bytes);
  if (most > idle / 2) most = idle / 2;
  if (idle >= 2 && y_bytes > 4 * v_bytes && most < 2) most = 2;
  int parts = split(most < 1 ? 1 : most > 8 ? 8 : (int)most, tile_waves(STAGES_VY));
  const size_t again = (size_t)(parts - 1) * tiles * l.n_proj * l.rank * l.in * 2;
  if (cpr > 4 && again > TILE_AGAIN) {
    const int groups = div_up(l.rank, 32);
    const dim3 gv(gx, l.n_proj * groups, slots(tiles * l.n_proj * groups, 2));
    const dim3 bv(64 * tile_waves(STAGES_V));
    if (xf32) k_lora_tile<STAGES_V, 4, true, false, false><<<gv, bv, 0, s>>>(a);
    else k_lora_tile<STAGES_V, 4, false, false, false><<<gv, bv, 0, s>>>(a);
    parts = 2 * N_CU / (tiles * l.n_proj);
    parts = split(parts < 1 ? 1 : parts, tile_waves(STAGES_Y));
    const dim3 gy(gx, l.n_proj * parts, slots(tiles * l.n_proj * parts, 2));
    if (cpr <= 6) launch_tile<STAGES_Y, 6, false>(a, gy, yf32, vec, s);
    else if (cpr <= 8) launch_tile<STAGES_Y, 8, false>(a, gy, yf32, vec, s);
    else if (cpr <= 12) launch_tile<STAGES_Y, 12, false>(a, gy, yf32, vec, s);
    else launch_tile<STAGES_Y, 16, false>(a, gy, yf32, vec, s);
    return hipGetLastError();
  }
  const dim3 grid(gx, l.n_proj * parts, slots(tiles * l.n_proj * parts, 4));
  if (cpr <= 1) launch_tile_vy<1>(a, grid, xf32, yf32, vec, s);
  else if (cpr <= 2) launch_tile_vy<2>(a, grid, xf32, yf32, vec, s);
  else if (cpr <= 4) launch_tile_vy<4>(a, grid, xf32, yf32, vec, s);
  else if (cpr <= 6) launch_tile_vy<6>(a, grid, xf32, yf32, vec, s);
  else if (cpr <= 8) launch_tile_vy<8>(a, grid, xf32, yf32, vec, s);
  else if (cpr <= 12) launch_tile_vy<12>(a, grid, xf32, yf32, vec, s);
  else launch_tile_vy<16>(a, grid, xf32, yf32, vec, s);
  return hipGetLastError();
}
