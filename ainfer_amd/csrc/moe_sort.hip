// moe_sort.hip - token rows into expert order and back (ainfer_moe_sort_rows,
// ainfer_moe_unpermute, ainfer_moe_unpermute_backward).
//
// The sort is a counting sort that keeps pairs of one expert in the order (token,
// slot): chunks of SORT_CHUNK pairs are counted per expert, and a chunk's first place
// for an expert is what all chunks have of smaller ones plus what earlier chunks
// have of the same.  Only integers are added in any order, so the result is one.
#include <algorithm>

#include "moe_common.h"
#include "moe_internal.h"
#include "moe_fp8_parts.h"

namespace {

constexpr int SORT_CHUNK = 1024;  // pairs of a chunk: 4 waves, 4 rounds of 64 each

// the expert of a pair, E for one that is dropped
__device__ __forceinline__ int expert_of(const int32_t *idx, int64_t i, int64_t n, int E) {
  const int e = i < n ? idx[i] : E;
  return (uint32_t)e < (uint32_t)E ? e : E;
}

// counts[chunk][E]
__global__ __launch_bounds__(256) void k_sort_count(const int32_t *idx, int64_t n, int E,
                                                    int32_t *counts) {
  __shared__ int32_t h[1024];
  for (int e = threadIdx.x; e < E; e += 256) h[e] = 0;
  __syncthreads();
  const int64_t c0 = (int64_t)blockIdx.x * SORT_CHUNK;
  for (int i = threadIdx.x; i < SORT_CHUNK; i += 256) {
    const int e = expert_of(idx, c0 + i, n, E);
    if (e < E) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += 256) counts[(int64_t)blockIdx.x * E + e] = h[e];
}

// pos of a chunk's pairs; the last workgroup writes offsets
__global__ __launch_bounds__(256) void k_sort_place(const int32_t *idx, int64_t n, int E,
                                                    const int32_t *counts, int chunks,
                                                    int32_t *offsets, int32_t *pos) {
  __shared__ int32_t at[4][1024];  // next place of each wave and expert
  __shared__ int32_t part[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t c0 = (int64_t)blockIdx.x * SORT_CHUNK + wave * (SORT_CHUNK / 4);
  for (int e = tid; e < 4 * 1024; e += 256) ((int32_t *)at)[e] = 0;
  __syncthreads();
  int ids[SORT_CHUNK / 256];
#pragma unroll
  for (int r = 0; r < SORT_CHUNK / 256; ++r) {
    ids[r] = expert_of(idx, c0 + r * 64 + lane, n, E);
    if (ids[r] < E) atomicAdd(&at[wave][ids[r]], 1);
  }
  // four neighbouring experts a thread: pairs of all chunks, and of those before this
  int all[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
  for (int c = 0; c < chunks; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = tid * 4 + i;
      const int v = e < E ? counts[(int64_t)c * E + e] : 0;
      all[i] += v;
      before[i] += c < (int)blockIdx.x ? v : 0;
    }
  const int mine = all[0] + all[1] + all[2] + all[3], incl = wave_scan_incl(mine);
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int first = incl - mine;
  for (int w = 0; w < wave; ++w) first += part[w];
  const bool last = blockIdx.x + 1 == gridDim.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    if (e < E) {
      if (last) offsets[e] = first;
      int p = first + before[i];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int c = at[w][e];
        at[w][e] = p;
        p += c;
      }
    }
    first += all[i];
    if (last && e == E - 1) offsets[E] = first;
  }
  __syncthreads();
  const int bits = 32 - __clz(E);  // of ids 0..E
#pragma unroll
  for (int r = 0; r < SORT_CHUNK / 256; ++r) {
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const bool on = ids[r] >> b & 1;
      const uint64_t m = __ballot(on);
      same &= on ? m : ~m;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), number = __popcll(same);
    const int64_t i = c0 + r * 64 + lane;
    const bool kept = ids[r] < E;
    const int p = kept ? at[wave][ids[r]] + rank : -1;
    if (i < n) pos[i] = p;
    __builtin_amdgcn_wave_barrier();
    if (kept && rank == 0) at[wave][ids[r]] = p + number;
    __builtin_amdgcn_wave_barrier();
  }
}

// Rows as they are: a lane takes 16 bytes of a token's row to its k places
// (SIZE: bytes of an element).
template <int SIZE>
__global__ __launch_bounds__(256) void k_move_rows(const uint8_t *x, int64_t xld,
                                                   const int32_t *pos, int T, int k, int H,
                                                   uint8_t *rows, int64_t rld) {
  constexpr int PER = 16 / SIZE;
  const int64_t per_row = (H + PER - 1) / PER, items = per_row * T;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t t = i / per_row;
    const int col = (int)(i - t * per_row) * PER;
    const uint8_t *src = x + (t * xld + col) * SIZE;
    const int left = H - col;
    if (left >= PER) {
      const u32x4 v = *(const u32x4_any *)src;
      for (int j = 0; j < k; ++j) {
        const int p = pos[t * k + j];
        if (p >= 0) *(u32x4_any *)(rows + (p * rld + col) * SIZE) = v;
      }
    } else {
      using el = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
      for (int j = 0; j < k; ++j) {
        const int p = pos[t * k + j];
        if (p >= 0)
          for (int d = 0; d < left; ++d) ((el *)(rows + (p * rld + col) * SIZE))[d] = ((const el *)src)[d];
      }
    }
  }
}

// Rows quantised once and written to their k places: 8 lanes a group of 128 columns.
template <bool F32>
__global__ __launch_bounds__(256) void k_move_quant(const void *x, int64_t xld, const int32_t *pos,
                                                    int T, int k, int H, int pow2, uint8_t *rows,
                                                    int64_t rld, float *sq) {
  const int G = (H + 127) / 128;
  const int64_t items = (int64_t)T * G * 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t t = i / (G * 8);
    const int col = (int)(i - t * (G * 8)) * 16;
    float v[16];
    if (col < H) {
      load_row<F32>(x, t * xld + col, v);
    } else {
#pragma unroll
      for (int d = 0; d < 16; ++d) v[d] = 0.0f;
    }
    float m = 0.0f;
#pragma unroll
    for (int d = 0; d < 16; ++d) m = max_skip_nan(m, fabsf(v[d]));
    const float s = fp8_scale(max_of_8_lanes(m), pow2);
    uint32_t w[4];
    fp8_codes(v, s, w);
    for (int j = 0; j < k; ++j) {
      const int64_t p = pos[t * k + j];
      if (p < 0) continue;
      if (col < H) *(u32x4 *)(rows + p * rld + col) = u32x4{w[0], w[1], w[2], w[3]};
      if ((threadIdx.x & 7) == 0) sq[p * G + col / 128] = s;
    }
  }
}

// y[t] = sum_j w[t][j] rows[pos[t][j]] (+ resid[t]), fp32 fma in slot order
template <bool RF32, bool YF32>
__global__ __launch_bounds__(256) void k_unpermute(const void *rows, int64_t rld, int N,
                                                   const int32_t *pos, const float *w, int T, int k,
                                                   int H, const void *resid, int64_t sld, void *y,
                                                   int64_t yld) {
  const int64_t per_row = (H + 7) / 8, items = per_row * T;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t t = i / per_row;
    const int col = (int)(i - t * per_row) * 8, left = H - col;
    float a[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8];
    for (int j = 0; j < k; ++j) {
      const int64_t p = pos[t * k + j];
      if ((uint64_t)p >= (uint64_t)N) continue;
      const float f = w ? w[t * k + j] : 1.0f;
      if (left >= 8) {
        load_row<RF32>(rows, p * rld + col, v);
#pragma unroll
        for (int d = 0; d < 8; ++d) a[d] = fmaf(f, v[d], a[d]);
      } else {
#pragma unroll
        for (int d = 0; d < 7; ++d)
          if (d < left) a[d] = fmaf(f, load_one<RF32>(rows, p * rld + col + d), a[d]);
      }
    }
    if (left >= 8) {
      if (resid) {
        load_row<YF32>(resid, t * sld + col, v);
#pragma unroll
        for (int d = 0; d < 8; ++d) a[d] += v[d];
      }
      store_row<YF32>(y, t * yld + col, a);
    } else {
#pragma unroll
      for (int d = 0; d < 7; ++d)
        if (d < left)
          store_one<YF32>(y, t * yld + col + d,
                          resid ? a[d] + load_one<YF32>(resid, t * sld + col + d) : a[d]);
    }
  }
}

// drows[pos[t][j]] = w[t][j] dy[t], dw[t][j] = <dy[t], rows[pos[t][j]]>: a workgroup
// takes a token; its threads' partial sums are added in a fixed order.
template <bool YF32, bool RF32>
__global__ __launch_bounds__(256) void k_unpermute_bwd(const void *dy, int64_t yld, const void *rows,
                                                       int64_t rld, int N, const int32_t *pos,
                                                       const float *w, int k, int H, void *drows,
                                                       int64_t dld, float *dw) {
  __shared__ float part[4];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x;
  for (int j = 0; j < k; ++j) {
    const int64_t p = pos[t * k + j];
    const bool there = (uint64_t)p < (uint64_t)N;
    const float f = w ? w[t * k + j] : 1.0f;
    float sum = 0.0f;
    for (int col = tid * 8; col < H && there; col += 256 * 8) {
      float g[8], v[8];
      if (H - col >= 8) {
        load_row<YF32>(dy, t * yld + col, g);
        if (dw) {
          load_row<RF32>(rows, p * rld + col, v);
#pragma unroll
          for (int d = 0; d < 8; ++d) sum = fmaf(g[d], v[d], sum);
        }
        if (drows) {
#pragma unroll
          for (int d = 0; d < 8; ++d) g[d] *= f;
          store_row<RF32>(drows, p * dld + col, g);
        }
      } else {
        for (int d = 0; d < H - col; ++d) {
          const float o = load_one<YF32>(dy, t * yld + col + d);
          if (dw) sum = fmaf(o, load_one<RF32>(rows, p * rld + col + d), sum);
          if (drows) store_one<RF32>(drows, p * dld + col + d, o * f);
        }
      }
    }
    if (dw) {
      for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
      if ((tid & 63) == 0) part[tid >> 6] = sum;
      __syncthreads();
      if (tid == 0) dw[t * k + j] = there ? (part[0] + part[1]) + (part[2] + part[3]) : 0.0f;
      __syncthreads();
    }
  }
}

}  // namespace

size_t sort_workspace_bytes(int T, int k, int E) {
  const size_t chunks = ((size_t)T * k + SORT_CHUNK - 1) / SORT_CHUNK;
  return (chunks * E * 4 + 255) & ~(size_t)255;
}

hipError_t launch_sort_rows(const ainfer_moe_sorting &d, const void *x, int64_t xld,
                            const int32_t *idx, int T, int32_t *offsets, int32_t *pos, void *rows,
                            int64_t rld, float *row_scales, void *ws, hipStream_t s) {
  const int k = d.top_k, E = d.n_experts, H = d.hidden;
  const int64_t n = (int64_t)T * k;
  const int chunks = (int)((n + SORT_CHUNK - 1) / SORT_CHUNK);
  int32_t *counts = (int32_t *)ws;
  if (chunks) k_sort_count<<<chunks, 256, 0, s>>>(idx, n, E, counts);
  // without tokens one workgroup writes E + 1 zeros
  k_sort_place<<<std::max(chunks, 1), 256, 0, s>>>(idx, n, E, counts, chunks, offsets, pos);
  if (!rows) return hipGetLastError();
  const bool f32 = d.x_dtype == AINFER_ACT_F32;
  auto grid = [](int64_t items) { return (int)std::min<int64_t>((items + 255) / 256, 8192); };
  if (d.fp8) {
    const int g = grid((int64_t)T * ((H + 127) / 128) * 8);
    const int pow2 = d.scale_kind == AINFER_FP8_SCALE_POW2;
    if (f32)
      k_move_quant<true><<<g, 256, 0, s>>>(x, xld, pos, T, k, H, pow2, (uint8_t *)rows, rld, row_scales);
    else
      k_move_quant<false><<<g, 256, 0, s>>>(x, xld, pos, T, k, H, pow2, (uint8_t *)rows, rld, row_scales);
  } else if (f32) {
    k_move_rows<4><<<grid((int64_t)T * ((H + 3) / 4)), 256, 0, s>>>((const uint8_t *)x, xld, pos, T, k, H,
                                                                   (uint8_t *)rows, rld);
  } else {
    k_move_rows<2><<<grid((int64_t)T * ((H + 7) / 8)), 256, 0, s>>>((const uint8_t *)x, xld, pos, T, k, H,
                                                                   (uint8_t *)rows, rld);
  }
  return hipGetLastError();
}

hipError_t launch_unpermute(const void *rows, int64_t rld, int rows_dtype, int N,
                            const int32_t *pos, const float *w, int T, int k, int H,
                            const void *resid, int64_t sld, void *y, int64_t yld, int y_dtype,
                            hipStream_t s) {
  const int64_t items = (int64_t)T * ((H + 7) / 8);
  const int grid = (int)std::min<int64_t>((items + 255) / 256, 8192);
  auto run = [&](auto kernel) {
    kernel<<<grid, 256, 0, s>>>(rows, rld, N, pos, w, T, k, H, resid, sld, y, yld);
  };
  const bool r32 = rows_dtype == AINFER_ACT_F32, y32 = y_dtype == AINFER_ACT_F32;
  if (r32) run(y32 ? k_unpermute<true, true> : k_unpermute<true, false>);
  else run(y32 ? k_unpermute<false, true> : k_unpermute<false, false>);
  return hipGetLastError();
}

hipError_t launch_unpermute_backward(const void *dy, int64_t yld, int y_dtype, const void *rows,
                                     int64_t rld, int rows_dtype, int N, const int32_t *pos,
                                     const float *w, int T, int k, int H, void *drows, int64_t dld,
                                     float *dw, hipStream_t s) {
  auto run = [&](auto kernel) {
    kernel<<<T, 256, 0, s>>>(dy, yld, rows, rld, N, pos, w, k, H, drows, dld, dw);
  };
  const bool r32 = rows_dtype == AINFER_ACT_F32, y32 = y_dtype == AINFER_ACT_F32;
  if (y32) run(r32 ? k_unpermute_bwd<true, true> : k_unpermute_bwd<true, false>);
  else run(r32 ? k_unpermute_bwd<false, true> : k_unpermute_bwd<false, false>);
  return hipGetLastError();
}
