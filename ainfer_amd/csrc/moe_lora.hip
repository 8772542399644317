// moe_lora.hip - low-rank adapters of many requests beside shared projections
// (ainfer_moe_lora_apply): y_p += scale_a (x A_a^T) B_a^T, a = the token's adapter.
//
// Tokens are taken in tiles of up to 16 neighbours, a column each of a
// v_mfma_f32_16x16x32_bf16; a tile runs once per distinct adapter in it, with the
// other tokens' columns ignored, so batches need no sorting: a batch of
// requests has one adapter per token (bound by reading A and B, where an empty
// column costs nothing), a prompt one adapter per tile.
//   k_lora_down  partial sums of v = x A^T over a part of K, to the workspace
//   k_lora_up    v = the sum of the parts, scaled; y += v B^T
// All products are exact: bf16 values enter the MFMA as they are, fp32 values as
// the sum of two or three bf16 (split_bf16).
#include "moe_common.h"
#include "moe_internal.h"

namespace {

constexpr int LT = 16;      // columns of a tile
constexpr int KB = 64;      // k of two MFMAs: 128 bytes of every bf16 row
constexpr int L_WAVES = 4;

struct LoraArgs {
  const void *x;
  const int32_t *ids, *ranks;
  const float *scales;
  const uint16_t *a[AINFER_LORA_MAX_PROJ], *b[AINFER_LORA_MAX_PROJ];
  void *y[AINFER_LORA_MAX_PROJ];
  int64_t y_ld[AINFER_LORA_MAX_PROJ], x_ld;
  int m[AINFER_LORA_MAX_PROJ];
  bool y_vec[AINFER_LORA_MAX_PROJ];  // y rows readable in 16-byte pieces
  float *part;    // [splits][P][T][R]
  int N, R, K, P, T;
  int tt;         // tokens per tile
  int splits;     // parts of K over workgroups
  int kw;         // blocks of KB per wave
  int units;      // 32-row units per wave of k_lora_up
};

// N values that sum to x, each exact in bf16 (x's bits from the top, 8 at a
// time: N = 3 holds all 24, N = 2 x to 2^-16), as fp32 with the low half clear.
// inf and NaN stay in the first.
template <int N>
__device__ __forceinline__ void split_bf16(float x, float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    x = x == s[i] ? 0.0f : x - s[i];
  }
}
// the high halves of two such values
__device__ __forceinline__ uint32_t pack_hi(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// ids of a tile's tokens, one per lane below tt; -1 = none
__device__ __forceinline__ int tile_ids(const LoraArgs &a, int t0, int lane) {
  int id = -1;
  if (lane < a.tt && t0 + lane < a.T) id = a.ids[t0 + lane];
  return id >= 0 && id < a.N ? id : -1;
}

// NRB: blocks of 16 rows of A.  A wave sums kw blocks of KB columns, the
// workgroup's four waves meet in LDS.
template <int NRB, bool XF32>
__global__ __launch_bounds__(64 * L_WAVES) void k_lora_down(LoraArgs a) {
  __shared__ f32x4 red[L_WAVES][NRB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = blockIdx.x * a.tt, p = blockIdx.z;
  const int id = tile_ids(a, t0, lane);
  uint64_t rem = __ballot(id >= 0);
  const int col = lane & 15, q = lane >> 4;
  const int row = min(t0 + min(col, a.tt - 1), a.T - 1);
  const int nb = (a.K + KB - 1) / KB;
  const int b0 = (blockIdx.y * L_WAVES + wave) * a.kw, b1 = min(b0 + a.kw, nb);
  const char *xr = (const char *)a.x + (size_t)row * a.x_ld * (XF32 ? 4 : 2);
  while (rem) {
    const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(rem));
    const uint64_t mask = __ballot(id == ad) & rem;
    rem &= ~mask;
    const uint16_t *A = a.a[p] + (size_t)ad * a.R * a.K;
    f32x4 acc[NRB];
#pragma unroll
    for (int r = 0; r < NRB; ++r) acc[r] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const uint16_t *ar[NRB];
#pragma unroll
    for (int r = 0; r < NRB; ++r) ar[r] = A + (size_t)min(r * 16 + col, a.R - 1) * a.K;
    for (int b = b0; b < b1; ++b) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = b * KB + q * 16 + h * 8;
        const bool in = k < a.K;  // K is a multiple of 8
        u32x4 af[NRB];
#pragma unroll
        for (int r = 0; r < NRB; ++r) af[r] = in ? *(const u32x4 *)(ar[r] + k) : (u32x4){0, 0, 0, 0};
        if constexpr (!XF32) {
          const u32x4 xf = in ? *(const u32x4 *)((const uint16_t *)xr + k) : (u32x4){0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < NRB; ++r) acc[r] = mfma_bf16_16x16x32(af[r], xf, acc[r]);
        } else {
          f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
          if (in) {
            v0 = *(const f32x4 *)((const float *)xr + k);
            v1 = *(const f32x4 *)((const float *)xr + k + 4);
          }
          u32x4 xf[3];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float lo[3], hi[3];
            split_bf16(i < 2 ? v0[2 * i] : v1[2 * i - 4], lo);
            split_bf16(i < 2 ? v0[2 * i + 1] : v1[2 * i - 3], hi);
#pragma unroll
            for (int s = 0; s < 3; ++s) xf[s][i] = pack_hi(lo[s], hi[s]);
          }
#pragma unroll
          for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int r = 0; r < NRB; ++r) acc[r] = mfma_bf16_16x16x32(af[r], xf[s], acc[r]);
        }
      }
    }
    __syncthreads();  // the previous adapter's sums are read
#pragma unroll
    for (int r = 0; r < NRB; ++r) red[wave][r][lane] = acc[r];
    __syncthreads();
    for (int r = wave; r < NRB; r += L_WAVES) {
      f32x4 v = red[0][r][lane];
#pragma unroll
      for (int w = 1; w < L_WAVES; ++w) v += red[w][r][lane];
      const int r0 = r * 16 + q * 4;
      if (((mask >> col) & 1) && r0 < a.R)
        *(f32x4 *)(a.part + (((size_t)blockIdx.y * a.P + p) * a.T + t0 + col) * a.R + r0) = v;
    }
  }
}

// NRK: blocks of 32 columns of B; NS: bf16 values that v enters as
template <int NRK, int NS, bool YF32>
__global__ __launch_bounds__(64 * L_WAVES) void k_lora_up(LoraArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = blockIdx.x * a.tt, p = blockIdx.z;
  const int M = a.m[p];
  const int u0 = (blockIdx.y * L_WAVES + wave) * a.units;
  if (u0 * 32 >= M) return;
  const int u1 = min(u0 + a.units, (M + 31) / 32);
  const int id = tile_ids(a, t0, lane);
  uint64_t rem = __ballot(id >= 0);
  const int col = lane & 15, q = lane >> 4;
  const int row = min(t0 + col, a.T - 1);
  while (rem) {
    const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(rem));
    const uint64_t mask = __ballot(id == ad) & rem;
    rem &= ~mask;
    int rank = a.R;
    if (a.ranks) rank = min(max(a.ranks[ad], 0), a.R);
    if (rank == 0) continue;
    const float scale = a.scales ? a.scales[ad] : 1.0f;
    const bool mine = (mask >> col) & 1;
    u32x4 vf[NRK][NS], keep[NRK];
#pragma unroll
    for (int rb = 0; rb < NRK; ++rb) {
      const int r0 = rb * 32 + q * 8;
      f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
      if (mine && r0 < a.R)
        for (int ks = 0; ks < a.splits; ++ks) {
          const float *v = a.part + (((size_t)ks * a.P + p) * a.T + row) * a.R + r0;
          s0 += *(const f32x4 *)v;
          s1 += *(const f32x4 *)(v + 4);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 2 * i;
        float lo[NS], hi[NS];
        split_bf16(r < rank ? (i < 2 ? s0[2 * i] : s1[2 * i - 4]) * scale : 0.0f, lo);
        split_bf16(r + 1 < rank ? (i < 2 ? s0[2 * i + 1] : s1[2 * i - 3]) * scale : 0.0f, hi);
#pragma unroll
        for (int s = 0; s < NS; ++s) vf[rb][s][i] = pack_hi(lo[s], hi[s]);
        keep[rb][i] = (r < rank ? 0xFFFFu : 0u) | (r + 1 < rank ? 0xFFFF0000u : 0u);
      }
    }
    const uint16_t *B = a.b[p] + (size_t)ad * M * a.R;
    for (int u = u0; u < u1; ++u) {
      // rows of B so that a lane ends with 8 consecutive ones of its token
      const int m0 = u * 32, mr = m0 + (col >> 2) * 8 + (col & 3);
      f32x4 acc[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint16_t *br = B + (size_t)min(mr + j * 4, M - 1) * a.R;
        acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int rb = 0; rb < NRK; ++rb) {
          const int r0 = rb * 32 + q * 8;
          u32x4 bf = {0, 0, 0, 0};
          if (r0 < rank) bf = *(const u32x4 *)(br + r0) & keep[rb];
#pragma unroll
          for (int s = 0; s < NS; ++s) acc[j] = mfma_bf16_16x16x32(bf, vf[rb][s], acc[j]);
        }
      }
      const int m = m0 + q * 8;
      if (!mine || m >= M) continue;
      const size_t at = (size_t)row * a.y_ld[p] + m;
      if (a.y_vec[p] && m + 8 <= M) {
        if constexpr (YF32) {
          f32x4 *y = (f32x4 *)((float *)a.y[p] + at);
          y[0] += acc[0];
          y[1] += acc[1];
        } else {
          u32x4 *y = (u32x4 *)((uint16_t *)a.y[p] + at);
          u32x4 v = *y;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lo = __uint_as_float(v[i] << 16) + acc[i / 2][2 * (i & 1)];
            const float hi = __uint_as_float(v[i] & 0xFFFF0000u) + acc[i / 2][2 * (i & 1) + 1];
            v[i] = (uint32_t)f32_to_bf16(lo) | ((uint32_t)f32_to_bf16(hi) << 16);
          }
          *y = v;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (m + i < M) {
            if constexpr (YF32) {
              ((float *)a.y[p])[at + i] += acc[i / 4][i & 3];
            } else {
              uint16_t *y = (uint16_t *)a.y[p] + at + i;
              *y = f32_to_bf16(bf16_to_f32(*y) + acc[i / 4][i & 3]);
            }
          }
      }
    }
  }
}

int div_up(int a, int b) { return (a + b - 1) / b; }

// Tokens per tile: one while a batch of requests (an adapter per token) fills
// the device with a workgroup each, 16 for prompts.
int tile_tokens(int T) { return T <= 64 ? 1 : T <= 256 ? 4 : LT; }

// Parts of K over workgroups: about LORA_WGS workgroups, a wave no less than one
// block of KB columns.
constexpr int LORA_WGS = 512, MAX_SPLITS = 16;
int k_splits(const ainfer_moe_lora &l, int T) {
  const int tiles = div_up(T, tile_tokens(T)) * l.n_proj;
  const int most = div_up(div_up(l.in, KB), L_WAVES);
  const int want = LORA_WGS / (tiles < LORA_WGS ? tiles : LORA_WGS);
  const int n = want < most ? want : most;
  return n < MAX_SPLITS ? n : MAX_SPLITS;
}

template <int NRK>
void launch_up(const LoraArgs &a, dim3 grid, bool yf32, hipStream_t s) {
  if (yf32)
    k_lora_up<NRK, 3, true><<<grid, 64 * L_WAVES, 0, s>>>(a);
  else
    k_lora_up<NRK, 2, false><<<grid, 64 * L_WAVES, 0, s>>>(a);
}
template <int NRB>
void launch_down(const LoraArgs &a, dim3 grid, bool xf32, hipStream_t s) {
  if (xf32)
    k_lora_down<NRB, true><<<grid, 64 * L_WAVES, 0, s>>>(a);
  else
    k_lora_down<NRB, false><<<grid, 64 * L_WAVES, 0, s>>>(a);
}

}  // namespace

// The parts of every call with up to max_tokens tokens: k_splits(T) * T is T
// itself, or at most LORA_WGS tiles' tokens, or MAX_SPLITS * T.
size_t lora_workspace_bytes(const ainfer_moe_lora &l, int max_tokens) {
  const size_t T = max_tokens, wide = (size_t)LORA_WGS * tile_tokens(max_tokens);
  const size_t split = T * MAX_SPLITS < wide ? T * MAX_SPLITS : wide;
  const size_t n = (T > split ? T : split) * l.n_proj * l.rank * sizeof(float);
  return (n + 255) & ~(size_t)255;
}

hipError_t launch_lora(const ainfer_moe_lora &l, const void *x, int64_t x_ld, const int32_t *ids,
                       int T, void *const *y, const int64_t *y_ld, void *ws, hipStream_t s) {
  LoraArgs a;
  a.x = x;
  a.ids = ids;
  a.ranks = l.ranks;
  a.scales = l.scales;
  a.x_ld = x_ld;
  a.part = (float *)ws;
  a.N = l.n_adapters;
  a.R = l.rank;
  a.K = l.in;
  a.P = l.n_proj;
  a.T = T;
  a.tt = tile_tokens(T);
  a.splits = k_splits(l, T);
  const int nb = div_up(l.in, KB);
  a.kw = div_up(nb, a.splits * L_WAVES);
  a.splits = div_up(nb, a.kw * L_WAVES);  // none empty
  const bool yf32 = l.y_dtype == AINFER_ACT_F32, xf32 = l.x_dtype == AINFER_ACT_F32;
  const int ysz = yf32 ? 4 : 2;
  int m_most = 1;
  for (int p = 0; p < AINFER_LORA_MAX_PROJ; ++p) {
    const bool on = p < l.n_proj;
    a.a[p] = on ? (const uint16_t *)l.a[p] : nullptr;
    a.b[p] = on ? (const uint16_t *)l.b[p] : nullptr;
    a.y[p] = on ? y[p] : nullptr;
    a.y_ld[p] = on ? y_ld[p] : 0;
    a.m[p] = on ? l.out[p] : 0;
    a.y_vec[p] = on && (uintptr_t)y[p] % 16 == 0 && (y_ld[p] * ysz) % 16 == 0;
    if (on && l.out[p] > m_most) m_most = l.out[p];
  }
  const int tiles = div_up(T, a.tt);
  const int nrb = div_up(l.rank, 16), nrk = div_up(l.rank, 32);
  const dim3 gd(tiles, a.splits, l.n_proj);
  if (nrb <= 1) launch_down<1>(a, gd, xf32, s);
  else if (nrb <= 2) launch_down<2>(a, gd, xf32, s);
  else if (nrb <= 4) launch_down<4>(a, gd, xf32, s);
  else launch_down<8>(a, gd, xf32, s);
  // rows of y over the workgroups
  const int units = div_up(m_most, 32);
  int per = div_up(units * tiles * l.n_proj, 4096);
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  a.units = per;
  const dim3 gu(tiles, div_up(units, per * L_WAVES), l.n_proj);
  if (nrk <= 1) launch_up<1>(a, gu, yf32, s);
  else if (nrk <= 2) launch_up<2>(a, gu, yf32, s);
  else launch_up<4>(a, gu, yf32, s);
  return hipGetLastError();
}
