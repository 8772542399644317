// moe_sort.hip - token rows into expert order and back (ainfer_moe_sort_rows,
// ainfer_moe_unpermute, ainfer_moe_unpermute_backward).
//
// The sort is a counting sort that keeps pairs of one expert in the order (token,
// slot): chunks of pairs are counted per expert, and a chunk's first place
// for an expert is what all chunks have of smaller ones plus what earlier chunks
// have of the same.  Only integers are added in any order, so the result is one.
//
// What bounds each, and us alone on the GPU: up to 2048 pairs one launch of latency (1 token of
// 4096 columns as codes 4.8; an empty launch takes 2.5); above, places are a launch of counting
// in LDS, or two of latency (65536 pairs of 64 experts 4.8 + 5.3), and the rows a pass
// at the speed of the memory: 4096 tokens of 2048 bf16 to 10 rows of codes 19.8, 103 MB; 8192
// of 4096 bf16 to 4 rows each 52, 6.4 TB/s.  Weighted sums of 4096 tokens, 10 rows of 2048 bf16
// 34.9, 5.3 TB/s; their gradients, 8 rows of 4096 bf16 108.5, 5.3.
#include <algorithm>

#include "moe_common.h"
#include "moe_internal.h"
#include "moe_fp8_parts.h"

namespace {

// A chunk is 4 waves x `rounds` of 64 pairs, 1024 pairs while that makes at most 256 chunks:
// every workgroup reads the counts of all of them.
int sort_rounds(int64_t n) { return 4 * (int)std::max<int64_t>(1, (n + 262143) / 262144); }

// the expert of a pair, E for one that is dropped
__device__ __forceinline__ int expert_of(const int32_t *idx, int64_t i, int64_t n, int E) {
  const int e = i < n ? idx[i] : E;
  return (uint32_t)e < (uint32_t)E ? e : E;
}

// counts[chunk][Ep], Ep = E rounded up to 4
__global__ __launch_bounds__(256) void k_sort_count(const int32_t *idx, int64_t n, int E, int Ep,
                                                    int rounds, int32_t *counts) {
  __shared__ int32_t h[1024];
  for (int e = threadIdx.x; e < Ep; e += 256) h[e] = 0;
  __syncthreads();
  const int64_t c0 = (int64_t)blockIdx.x * rounds * 256;
  for (int r0 = 0; r0 < rounds; r0 += 4) {
    int ids[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) ids[r] = expert_of(idx, c0 + (r0 + r) * 256 + threadIdx.x, n, E);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (ids[r] < E) atomicAdd(&h[ids[r]], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < Ep; e += 256) counts[(int64_t)blockIdx.x * Ep + e] = h[e];
}

// The places of a chunk's pairs: waves 0 to 3 of a workgroup have them in order, `rounds` of
// 64 each (from c0, the wave's first).
struct ChunkPlaces {
  int32_t at[4][1024];  // next place of each wave and expert
};
__device__ __forceinline__ void count_chunk(ChunkPlaces &c, const int32_t *idx, int64_t c0,
                                            int64_t n, int E, int rounds) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave >= 4) return;
  for (int r0 = 0; r0 < rounds; r0 += 4) {
    int ids[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      ids[r] = r0 + r < rounds ? expert_of(idx, c0 + (r0 + r) * 64 + lane, n, E) : E;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (ids[r] < E) atomicAdd(&c.at[wave][ids[r]], 1);
  }
}
// the four waves' counts of expert e become their first places
__device__ __forceinline__ void first_places(ChunkPlaces &c, int e, int first) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int n = c.at[w][e];
    c.at[w][e] = first;
    first += n;
  }
}
__device__ __forceinline__ void place_chunk(ChunkPlaces &c, const int32_t *idx, int64_t c0,
                                            int64_t n, int E, int rounds, int32_t *pos) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave >= 4) return;
  const int bits = 32 - __clz(E);  // of ids 0..E
  for (int r0 = 0; r0 < rounds; r0 += 4) {
    int ids[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      ids[r] = r0 + r < rounds ? expert_of(idx, c0 + (r0 + r) * 64 + lane, n, E) : E;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r0 + r >= rounds) break;
      uint64_t same = ~0ull;  // the lanes with this lane's id
      for (int b = 0; b < bits; ++b) {
        const bool on = ids[r] >> b & 1;
        const uint64_t m = __ballot(on);
        same &= on ? m : ~m;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1)), number = __popcll(same);
      const int64_t i = c0 + (r0 + r) * 64 + lane;
      const bool kept = ids[r] < E;
      const int p = kept ? c.at[wave][ids[r]] + rank : -1;
      if (i < n) pos[i] = p;
      __builtin_amdgcn_wave_barrier();
      if (kept && rank == 0) c.at[wave][ids[r]] = p + number;
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// pos of a chunk's pairs; the last workgroup writes offsets.  The chunks' counts are read in
// columns of four experts by groups of threads that take every so many-th chunk, several
// loads at once (one thread for each column, one chunk after the other: 18.5 instead of
// 6.9 us for 40 chunks of 512 experts).
__global__ __launch_bounds__(256) void k_sort_place(const int32_t *idx, int64_t n, int E, int Ep,
                                                    int rounds, const int32_t *counts, int chunks,
                                                    int32_t *offsets, int32_t *pos) {
  __shared__ ChunkPlaces places;
  __shared__ int32_t all[1024], before[1024];  // pairs of every chunk, and of those before this
  __shared__ int32_t part[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t c0 = ((int64_t)blockIdx.x * 4 + wave) * rounds * 64;
  for (int e = tid; e < 1024; e += 256) {
    all[e] = before[e] = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) places.at[w][e] = 0;
  }
  __syncthreads();
  count_chunk(places, idx, c0, n, E, rounds);
  const int columns = Ep / 4, groups = max(1, 256 / columns), mine = tid / columns;
  if (mine < groups) {
    const int e = (tid - mine * columns) * 4;
    int4 sum = {0, 0, 0, 0}, low = {0, 0, 0, 0};
    const int32_t *p = counts + e;
    auto add = [&](int4 v, int c) {
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      if (c < (int)blockIdx.x) low.x += v.x, low.y += v.y, low.z += v.z, low.w += v.w;
    };
    int c = mine;
    for (; c + 7 * groups < chunks; c += 8 * groups) {
      int4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = *(const int4 *)(p + (int64_t)(c + u * groups) * Ep);
#pragma unroll
      for (int u = 0; u < 8; ++u) add(v[u], c + u * groups);
    }
    if (c < chunks) {  // up to seven more, the last one again instead of none
      int4 v[7];
#pragma unroll
      for (int u = 0; u < 7; ++u)
        v[u] = *(const int4 *)(p + (int64_t)min(c + u * groups, chunks - 1) * Ep);
#pragma unroll
      for (int u = 0; u < 7; ++u)
        if (c + u * groups < chunks) add(v[u], c + u * groups);
    }
    const int32_t s4[4] = {sum.x, sum.y, sum.z, sum.w}, l4[4] = {low.x, low.y, low.z, low.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      atomicAdd(&all[e + i], s4[i]);
      atomicAdd(&before[e + i], l4[i]);
    }
  }
  __syncthreads();
  int own[4], total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) total += own[i] = all[tid * 4 + i];
  const int incl = wave_scan_incl(total);
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int first = incl - total;
  for (int w = 0; w < wave; ++w) first += part[w];
  const bool last = blockIdx.x + 1 == gridDim.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    if (e < E) {
      if (last) offsets[e] = first;
      first_places(places, e, first + before[e]);
    }
    first += own[i];
    if (last && e == E - 1) offsets[E] = first;
  }
  __syncthreads();
  place_chunk(places, idx, c0, n, E, rounds, pos);
}

// Up to SORT_OWN pairs, in one launch: a workgroup of 16 waves counts all pairs itself, all
// of them in the low half of a word and those of earlier chunks in the high half, four words
// an expert for neighbouring lanes (pairs that all name one expert would take 64 turns of
// the LDS at one word).  Its chunk is 256 pairs, placed by four of its waves.  Counting takes
// 0.1 us for 1000 pairs, in rounds of 16384.  us of this launch, and of two that share the counts:
// 2400 pairs of 64 experts 7.4, 9.3 (each with a launch of short rows); 16000 8.6, 11.1.  Three
// rounds are the most: in a graph, ids spread evenly, 49152 pairs of 16 experts 7.9, 7.7, of 64 7.7,
// 7.9, of 512 6.9, 9.8; 53248 8.9, 7.8; 8.6, 7.9; 7.8, 10.2.  Busy experts cost this launch more:
// 49152 by a power law 10.2, 7.9; 8.8, 8.0; 7.7, 9.8; all of one 14.4, 9.0.
constexpr int SORT_OWN = 3 * 16384;  // 16 bits hold it
typedef int32_t i32x4_any __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(1024) void k_sort_own(const int32_t *idx, int n, int E,
                                                   int32_t *offsets, int32_t *pos) {
  constexpr int COPY = 1024 + 8;
  __shared__ ChunkPlaces places;
  __shared__ uint32_t h[4 * COPY];
  __shared__ int32_t part[16];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int first_pair = blockIdx.x * 256;
  for (int i = tid; i < 4 * COPY; i += 1024) h[i] = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) places.at[w][tid] = 0;
  __syncthreads();
  count_chunk(places, idx, first_pair + wave * 64, n, E, 1);
  uint32_t *mine = h + (lane & 3) * COPY;
  for (int i = tid * 4; i < n; i += 4 * 4096) {
    i32x4_any v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = i + u * 4096;
      v[u] = i32x4_any{-1, -1, -1, -1};
      if (at + 4 <= n) {
        v[u] = *(const i32x4_any *)(idx + at);
      } else {
#pragma unroll
        for (int d = 0; d < 3; ++d)
          if (at + d < n) v[u][d] = idx[at + d];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if ((uint32_t)v[u][d] < (uint32_t)E)
          atomicAdd(&mine[v[u][d]], i + u * 4096 + d < first_pair ? 0x10001u : 1u);
  }
  __syncthreads();
  const uint32_t c = (h[tid] + h[COPY + tid]) + (h[2 * COPY + tid] + h[3 * COPY + tid]);
  const int own = c & 0xFFFF, incl = wave_scan_incl(own);
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int first = incl - own;
  for (int w = 0; w < wave; ++w) first += part[w];
  if (tid < E) first_places(places, tid, first + (int)(c >> 16));
  if (blockIdx.x + 1 == gridDim.x && tid < E) {
    offsets[tid] = first;
    if (tid == E - 1) offsets[E] = first + own;
  }
  __syncthreads();
  place_chunk(places, idx, first_pair + wave * 64, n, E, 1, pos);
}

// Few pairs (SORT_FEW at most; 4000 of them 16.1 instead of 12.7 us): everything in one
// launch.  Workgroup (t, y) takes token t and every gridDim.y-th part of its columns, and
// counts the smaller pairs for the token's k itself; workgroup (T, 0) writes offsets.  MODE:
// bytes of an element of rows that are moved as they are, or 8 (bf16) and 9 (fp32) for rows
// that are quantised; 0 for none.
constexpr int SORT_FEW = 2048;

template <int MODE>
__global__ __launch_bounds__(256) void k_sort_few(const int32_t *idx, int T, int k, int E,
                                                  int32_t *offsets, int32_t *pos, const void *x,
                                                  int64_t xld, int H, int pow2, uint8_t *rows,
                                                  int64_t rld, float *sq) {
  __shared__ int32_t h[1024];
  __shared__ int32_t sum[4][32];
  __shared__ int32_t at[32];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = T * k;
  int ids[SORT_FEW / 256];
#pragma unroll
  for (int r = 0; r < SORT_FEW / 256; ++r) {
    ids[r] = E;
    if (r * 256 < n) ids[r] = expert_of(idx, r * 256 + tid, n, E);
  }
  const int t = blockIdx.x;
  if (t == T) {
    if (blockIdx.y) return;
    for (int e = tid; e < 1024; e += 256) h[e] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_FEW / 256; ++r)
      if (ids[r] < E) atomicAdd(&h[ids[r]], 1);
    __syncthreads();
    int own[4], total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) total += own[i] = h[tid * 4 + i];
    const int incl = wave_scan_incl(total);
    if (lane == 63) at[wave] = incl;
    __syncthreads();
    int first = incl - total;
    for (int w = 0; w < wave; ++w) first += at[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = tid * 4 + i;
      if (e < E) offsets[e] = first;
      first += own[i];
      if (e == E - 1) offsets[E] = first;
    }
    return;
  }
  // the first columns are on their way while the pairs are counted
  constexpr bool QUANT = MODE >= 8, F32 = MODE == 9;
  constexpr int PER = QUANT ? 16 : MODE ? 16 / MODE : 1;
  const int pieces = QUANT ? (H + 127) / 128 * 8 : MODE ? (H + PER - 1) / PER : 0;
  int c = blockIdx.y * 256 + tid;
  float v[16];
  u32x4 raw = {0, 0, 0, 0};
  auto load = [&]() {
    if constexpr (QUANT) {
      if (c < pieces && c * 16 < H) {
        load_row<F32>(x, t * xld + c * 16, v);
      } else {
#pragma unroll
        for (int d = 0; d < 16; ++d) v[d] = 0.0f;
      }
    } else if constexpr (MODE != 0) {
      if (c < pieces && H >= PER)
        raw = *(const u32x4_any *)((const uint8_t *)x + (t * xld + min(c * PER, H - PER)) * MODE);
    }
  };
  load();
  const int owns = lane < k ? expert_of(idx, t * k + lane, n, E) : E;  // lane j: the token's j-th
  for (int j = 0; j < k; ++j) {
    const int own = __builtin_amdgcn_readlane(owns, j);
    int smaller = 0;
#pragma unroll
    for (int r = 0; r < SORT_FEW / 256; ++r)
      if (r * 256 < n)
        smaller += __popcll(__ballot(ids[r] < own || (ids[r] == own && r * 256 + tid < t * k + j)));
    if (lane == 0) sum[wave][j] = smaller;
  }
  __syncthreads();
  if (tid < k) {
    const int p = owns < E ? (sum[0][tid] + sum[1][tid]) + (sum[2][tid] + sum[3][tid]) : -1;
    at[tid] = p;
    if (blockIdx.y == 0) pos[t * k + tid] = p;
  }
  __syncthreads();
  if constexpr (MODE != 0) {
    for (; c - tid < pieces; c += gridDim.y * 256, load()) {
      if constexpr (QUANT) {
        float m = 0.0f;
#pragma unroll
        for (int d = 0; d < 16; ++d) m = max_skip_nan(m, fabsf(v[d]));
        const float s = fp8_scale(max_of_8_lanes(m), pow2);
        if (c >= pieces) continue;
        uint32_t w[4];
        fp8_codes(v, s, w);
        const int G = pieces / 8;
        for (int j = 0; j < k; ++j) {
          const int64_t p = at[j];
          if (p < 0) continue;
          if (c * 16 < H) *(u32x4 *)(rows + p * rld + c * 16) = u32x4{w[0], w[1], w[2], w[3]};
          if ((tid & 7) == 0) sq[p * G + c / 8] = s;
        }
      } else {
        if (c >= pieces) continue;
        const int col = min(c * PER, H - PER);  // the last piece: the row's last 16 bytes
        for (int j = 0; j < k; ++j) {
          const int64_t p = at[j];
          if (p < 0) continue;
          if (H >= PER) {
            *(u32x4_any *)(rows + (p * rld + col) * MODE) = raw;
          } else {
            using el = typename std::conditional<MODE == 4, uint32_t, uint16_t>::type;
            for (int d = 0; d < H; ++d) ((el *)rows)[p * rld + d] = ((const el *)x)[t * xld + d];
          }
        }
      }
    }
  }
}

// Rows as they are: a lane takes 16 bytes of a token's row to its k places (SIZE: bytes of an
// element; the last piece of a row is its last 16), past the caches (ordinary stores: 68 instead
// of 51 us for 8192 rows of 4096 bf16, half of 8 places each; 268 MB written).
template <int SIZE>
__global__ __launch_bounds__(256) void k_move_rows(const uint8_t *x, int64_t xld,
                                                   const int32_t *pos, int T, int k, int H,
                                                   uint8_t *rows, int64_t rld) {
  constexpr int PER = 16 / SIZE;
  const int64_t per_row = (H + PER - 1) / PER, items = per_row * T;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t t = i / per_row;
    if (H >= PER) {
      const int col = min((int)(i - t * per_row) * PER, H - PER);
      const u32x4 v = *(const u32x4_any *)(x + (t * xld + col) * SIZE);
      for (int j = 0; j < k; ++j) {
        const int p = pos[t * k + j];
        if (p >= 0) __builtin_nontemporal_store(v, (u32x4_any *)(rows + (p * rld + col) * SIZE));
      }
    } else {
      using el = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
      for (int j = 0; j < k; ++j) {
        const int p = pos[t * k + j];
        if (p >= 0)
          for (int d = 0; d < H; ++d) ((el *)rows)[p * rld + d] = ((const el *)x)[t * xld + d];
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
      if (col < H)
        __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, (u32x4 *)(rows + p * rld + col));
      if ((threadIdx.x & 7) == 0) sq[p * G + col / 128] = s;
    }
  }
}

// Eight values as they are in memory.  bf16 rows are read past the caches: a row is read once
// (ordinary loads: 40.8 instead of 35.6 us for 4096 tokens, 10 rows of 2048 each).  fp32 rows
// are not: a lane's two pieces are two loads, which would fetch each line twice.
template <bool F32>
struct Eight {
  u32x4 v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t at) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = *(const u32x4_any *)((const float *)p + at + 4 * i);
    } else {
      v[0] = __builtin_nontemporal_load((const u32x4_any *)((const uint16_t *)p + at));
    }
  }
  __device__ __forceinline__ float get(int d) const {
    if constexpr (F32) return __uint_as_float(v[d / 4][d % 4]);
    else return __uint_as_float(d & 1 ? v[0][d / 2] & 0xFFFF0000u : v[0][d / 2] << 16);
  }
};

// y[t] = sum_j w[t][j] rows[pos[t][j]] (+ resid[t]), fp32 fma in slot order.  A lane takes
// eight columns of a token; two rows are on their way at a time.  The last lane of a row that
// is no multiple of 8 reads the rows' last eight columns (column by column: 219 tokens, 5 rows of
// 5353, 11.6 instead of 7.5 us).
template <bool RF32, bool YF32>
__global__ __launch_bounds__(256) void k_unpermute(const void *rows, int64_t rld, int N,
                                                   const int32_t *pos, const float *w, int T, int k,
                                                   int H, const void *resid, int64_t sld, void *y,
                                                   int64_t yld) {
  constexpr int U = 2;
  const int64_t per_row = (H + 7) / 8, items = per_row * T;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t t = i / per_row;
    const int col = (int)(i - t * per_row) * 8, left = H - col;
    float a[8] = {0, 0, 0, 0, 0, 0, 0, 0}, r[8];
    if (H >= 8) {
      const int at = min(col, H - 8);  // the last lane of a row takes its last eight columns
      for (int j0 = 0; j0 < k; j0 += U) {
        Eight<RF32> v[U];
        float f[U];
        bool there[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          there[u] = false;
          if (j0 + u < k) {
            const int64_t p = pos[t * k + j0 + u];
            there[u] = (uint64_t)p < (uint64_t)N;
            if (there[u]) {
              f[u] = w ? w[t * k + j0 + u] : 1.0f;
              v[u].load(rows, p * rld + at);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (there[u]) {
#pragma unroll
            for (int d = 0; d < 8; ++d) a[d] = fmaf(f[u], v[u].get(d), a[d]);
          }
      }
      if (left >= 8) {
        if (resid) {
          load_row<YF32>(resid, t * sld + col, r);
#pragma unroll
          for (int d = 0; d < 8; ++d) a[d] += r[d];
        }
        store_row<YF32>(y, t * yld + col, a);
      } else {  // its own columns alone: resid may be y
#pragma unroll
        for (int d = 1; d < 8; ++d)
          if (at + d >= col && resid) a[d] += load_one<YF32>(resid, t * sld + at + d);
#pragma unroll
        for (int d = 1; d < 8; ++d)
          if (at + d >= col) store_one<YF32>(y, t * yld + at + d, a[d]);
      }
    } else {
      for (int j = 0; j < k; ++j) {
        const int64_t p = pos[t * k + j];
        if ((uint64_t)p >= (uint64_t)N) continue;
        const float f = w ? w[t * k + j] : 1.0f;
#pragma unroll
        for (int d = 0; d < 7; ++d)
          if (d < left) a[d] = fmaf(f, load_one<RF32>(rows, p * rld + d), a[d]);
      }
#pragma unroll
      for (int d = 0; d < 7; ++d)
        if (d < left)
          store_one<YF32>(y, t * yld + d,
                          resid ? a[d] + load_one<YF32>(resid, t * sld + d) : a[d]);
    }
  }
}

// drows[pos[t][j]] = w[t][j] dy[t], dw[t][j] = <dy[t], rows[pos[t][j]]>: workgroup (t, y) takes
// pairs 2 y and 2 y + 1 of token t; its threads' partial sums are added in one order.  (One
// workgroup for all of a token's pairs: 219 tokens of 5 pairs, 5353 columns, 16.7 instead of
// 9.8 us; 16 of 8, 2048, 6.8 instead of 3.3; 4096 of 8, 4096, 111 instead of 108.5.)
// A lane takes eight columns; the last lane of a row that is no multiple of 8 takes the row's
// last eight, of which it writes all (values that its neighbour writes too) and sums its own.
template <bool YF32, bool RF32>
__global__ __launch_bounds__(256) void k_unpermute_bwd(const void *dy, int64_t yld, const void *rows,
                                                       int64_t rld, int N, const int32_t *pos,
                                                       const float *w, int k, int H, void *drows,
                                                       int64_t dld, float *dw) {
  constexpr int J = 2;
  __shared__ float part[J][4];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, j0 = J * blockIdx.y;
  int64_t p[J];
  float f[J], sum[J];
#pragma unroll
  for (int u = 0; u < J; ++u) {
    p[u] = j0 + u < k ? pos[t * k + j0 + u] : -1;
    if (p[u] >= N) p[u] = -1;
    f[u] = w && j0 + u < k ? w[t * k + j0 + u] : 1.0f;
    sum[u] = 0.0f;
  }
  for (int own = tid * 8; own < H; own += 256 * 8) {
    if (H >= 8) {
      const int col = min(own, H - 8);
      Eight<RF32> v[J];
      if (dw) {
#pragma unroll
        for (int u = 0; u < J; ++u)
          if (p[u] >= 0) v[u].load(rows, p[u] * rld + col);
      }
      float g[8];
      load_row<YF32>(dy, t * yld + col, g);
      if (drows) {
#pragma unroll
        for (int u = 0; u < J; ++u)
          if (p[u] >= 0) {
            float o[8];
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d] = g[d] * f[u];
            store_row<RF32, 8, !RF32>(drows, p[u] * dld + col, o);
          }
      }
      if (dw) {
#pragma unroll
        for (int u = 0; u < J; ++u) {
          if (p[u] < 0) continue;
          if (col == own) {
#pragma unroll
            for (int d = 0; d < 8; ++d) sum[u] = fmaf(g[d], v[u].get(d), sum[u]);
          } else {
#pragma unroll
            for (int d = 1; d < 8; ++d)
              if (col + d >= own) sum[u] = fmaf(g[d], v[u].get(d), sum[u]);
          }
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < J; ++u)
        if (p[u] >= 0)
          for (int d = 0; d < H; ++d) {
            const float o = load_one<YF32>(dy, t * yld + d);
            if (dw) sum[u] = fmaf(o, load_one<RF32>(rows, p[u] * rld + d), sum[u]);
            if (drows) store_one<RF32>(drows, p[u] * dld + d, o * f[u]);
          }
    }
  }
  if (dw) {
#pragma unroll
    for (int u = 0; u < J; ++u) {
      for (int o = 32; o; o >>= 1) sum[u] += __shfl_xor(sum[u], o, 64);
      if ((tid & 63) == 0) part[u][wave] = sum[u];
    }
    __syncthreads();
    if (tid < J && j0 + tid < k)
      dw[t * k + j0 + tid] = (part[tid][0] + part[tid][1]) + (part[tid][2] + part[tid][3]);
  }
}

}  // namespace

size_t sort_workspace_bytes(int T, int k, int E) {
  // (fewer tokens than T never have more chunks than T and 256)
  const size_t chunks = std::min<size_t>(256, ((size_t)T * k + 1023) / 1024);
  return (chunks * ((E + 3) & ~3) * 4 + 255) & ~(size_t)255;
}

hipError_t launch_sort_rows(const ainfer_moe_sorting &d, const void *x, int64_t xld,
                            const int32_t *idx, int T, int32_t *offsets, int32_t *pos, void *rows,
                            int64_t rld, float *row_scales, void *ws, hipStream_t s) {
  const int k = d.top_k, E = d.n_experts, H = d.hidden;
  const int64_t n = (int64_t)T * k;
  const int rounds = sort_rounds(n), chunks = (int)((n + rounds * 256 - 1) / (rounds * 256));
  const int pow2 = d.scale_kind == AINFER_FP8_SCALE_POW2;
  const bool f32 = d.x_dtype == AINFER_ACT_F32;
  if (n <= SORT_FEW) {
    // columns of a token over several workgroups while there are few of them
    const int pieces = !rows ? 1 : d.fp8 ? (H + 15) / 16 : (H + (f32 ? 3 : 7)) / (f32 ? 4 : 8);
    const int parts = std::max(1, std::min((pieces + 255) / 256, 256 / std::max(T, 1)));
    auto few = [&](auto kernel) {
      return enqueue(kernel, dim3(T + 1, parts), 256, s, idx, T, k, E, offsets, pos, x, xld, H, pow2,
                     (uint8_t *)rows, rld, row_scales);
    };
    if (!rows) return few(k_sort_few<0>);
    if (d.fp8) return few(f32 ? k_sort_few<9> : k_sort_few<8>);
    return few(f32 ? k_sort_few<4> : k_sort_few<2>);
  }
  hipError_t rc;
  if (n <= SORT_OWN) {
    rc = enqueue(k_sort_own, (int)((n + 255) / 256), 1024, s, idx, (int)n, E, offsets, pos);
  } else {
    int32_t *counts = (int32_t *)ws;
    const int Ep = (E + 3) & ~3;
    rc = enqueue(k_sort_count, chunks, 256, s, idx, n, E, Ep, rounds, counts);
    if (rc == hipSuccess)
      rc = enqueue(k_sort_place, chunks, 256, s, idx, n, E, Ep, rounds, counts, chunks, offsets, pos);
  }
  if (rc != hipSuccess || !rows) return rc;
  auto grid = [](int64_t items) { return (int)std::min<int64_t>((items + 255) / 256, 8192); };
  if (d.fp8)
    return enqueue(f32 ? k_move_quant<true> : k_move_quant<false>,
                   grid((int64_t)T * ((H + 127) / 128) * 8), 256, s, x, xld, pos, T, k, H, pow2,
                   (uint8_t *)rows, rld, row_scales);
  return enqueue(f32 ? k_move_rows<4> : k_move_rows<2>, grid((int64_t)T * (f32 ? (H + 3) / 4 : (H + 7) / 8)),
                 256, s, (const uint8_t *)x, xld, pos, T, k, H, (uint8_t *)rows, rld);
}

hipError_t launch_unpermute(const void *rows, int64_t rld, int rows_dtype, int N,
                            const int32_t *pos, const float *w, int T, int k, int H,
                            const void *resid, int64_t sld, void *y, int64_t yld, int y_dtype,
                            hipStream_t s) {
  const int64_t items = (int64_t)T * ((H + 7) / 8);
  const int grid = (int)std::min<int64_t>((items + 255) / 256, 8192);
  auto run = [&](auto kernel) {
    return enqueue(kernel, grid, 256, s, rows, rld, N, pos, w, T, k, H, resid, sld, y, yld);
  };
  const bool r32 = rows_dtype == AINFER_ACT_F32, y32 = y_dtype == AINFER_ACT_F32;
  if (r32) return run(y32 ? k_unpermute<true, true> : k_unpermute<true, false>);
  return run(y32 ? k_unpermute<false, true> : k_unpermute<false, false>);
}

hipError_t launch_unpermute_backward(const void *dy, int64_t yld, int y_dtype, const void *rows,
                                     int64_t rld, int rows_dtype, int N, const int32_t *pos,
                                     const float *w, int T, int k, int H, void *drows, int64_t dld,
                                     float *dw, hipStream_t s) {
  auto run = [&](auto kernel) {
    return enqueue(kernel, dim3(T, (k + 1) / 2), 256, s, dy, yld, rows, rld, N, pos, w, k, H, drows, dld,
                   dw);
  };
  const bool r32 = rows_dtype == AINFER_ACT_F32, y32 = y_dtype == AINFER_ACT_F32;
  if (y32) return run(r32 ? k_unpermute_bwd<true, true> : k_unpermute_bwd<true, false>);
  return run(r32 ? k_unpermute_bwd<false, true> : k_unpermute_bwd<false, false>);
}
