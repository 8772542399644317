// moe_silu.hip - the gated activation between an MLP's projections
// (ainfer_moe_silu_mul): act = g / (1 + exp(-g)) * u, rows of any pitch.
// One pass, bound by memory: two inputs read, one output written.  4096 x 17408 bf16
// 84.6 us, 5.05 TB/s (a large copy reaches 5.13), 4609 x 7139 fp32 73; 16 x 1024 2.5 us,
// which an empty launch takes too.  And its gradient (ainfer_moe_silu_mul_backward): three
// inputs, two outputs, bound the same way; 32768 x 1024 bf16 57 us, 5.9 TB/s.
#include "moe_common.h"
#include "moe_internal.h"

namespace {

// vectors at any address of their elements: rows of an odd length or pitch are read
// in 16-byte pieces as well (the hardware's unaligned global accesses)
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

template <bool F32>
__device__ __forceinline__ void load8(const void *p, int64_t at, float (&v)[8]) {
  if constexpr (F32) {
    const f32x4 a = *(const f32x4_any *)((const float *)p + at);
    const f32x4 b = *(const f32x4_any *)((const float *)p + at + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    const u32x4 a = *(const u32x4_any *)((const uint16_t *)p + at);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = __uint_as_float(i & 1 ? a[i / 2] & 0xFFFF0000u : a[i / 2] << 16);
  }
}
template <bool F32>
__device__ __forceinline__ float load1(const void *p, int64_t at) {
  return F32 ? ((const float *)p)[at] : bf16_to_f32(((const uint16_t *)p)[at]);
}

// a lane takes 8 values of a row, the last lane of a row what is left of it
template <bool IF32, bool OF32>
__global__ __launch_bounds__(256) void k_silu_rows(const void *g, int64_t gld, const void *u,
                                                   int64_t uld, void *y, int64_t yld, int64_t n8,
                                                   int64_t per_row, int64_t I) {
  for (int64_t c = blockIdx.x * 256ll + threadIdx.x; c < n8; c += gridDim.x * 256ll) {
    int64_t row = 0;
    if (per_row != n8)  // a division of 32 bits where that will do
      row = n8 >> 32 ? c / per_row : (int64_t)((uint32_t)c / (uint32_t)per_row);
    const int64_t col = (c - row * per_row) * 8;
    const int64_t gat = row * gld + col, uat = row * uld + col, at = row * yld + col;
    if (I - col >= 8) {
      float gv[8], uv[8], o[8];
      load8<IF32>(g, gat, gv);
      load8<IF32>(u, uat, uv);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = silu_mul(gv[i], uv[i]);
      if constexpr (OF32) {
        float *p = (float *)y + at;
        *(f32x4_any *)p = (f32x4){o[0], o[1], o[2], o[3]};
        *(f32x4_any *)(p + 4) = (f32x4){o[4], o[5], o[6], o[7]};
      } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = (uint32_t)f32_to_bf16(o[2 * i]) | ((uint32_t)f32_to_bf16(o[2 * i + 1]) << 16);
        *(u32x4_any *)((uint16_t *)y + at) = w;
      }
    } else {
      for (int i = 0; i < (int)(I - col); ++i) {
        const float o = silu_mul(load1<IF32>(g, gat + i), load1<IF32>(u, uat + i));
        if constexpr (OF32) ((float *)y)[at + i] = o;
        else ((uint16_t *)y)[at + i] = f32_to_bf16(o);
      }
    }
  }
}

// d_gate = d * up * sig (1 + gate (1 - sig)), d_up = d * gate * sig, sig = 1 / (1 + exp(-gate))
__device__ __forceinline__ void silu_grad(float d, float g, float u, float &dg, float &du) {
  const float sig = 1.0f / (1.0f + expf(-g));
  dg = d * u * (sig * (1.0f + g * (1.0f - sig)));
  du = d * (g * sig);
}

// eight values read and written past the caches where that is one piece of 16 bytes a lane
// (32768 x 1024 bf16: 57 us, 63 with ordinary accesses; with fp32's two pieces a lane
// 177 instead of 155 us for 40000 x 1000)
template <bool F32>
__device__ __forceinline__ void load8_once(const void *p, int64_t at, float (&v)[8]) {
  if constexpr (F32) {
    load8<F32>(p, at, v);
  } else {
    const u32x4 a = __builtin_nontemporal_load((const u32x4_any *)((const uint16_t *)p + at));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = __uint_as_float(i & 1 ? a[i / 2] & 0xFFFF0000u : a[i / 2] << 16);
  }
}
template <bool F32>
__device__ __forceinline__ void store8_once(void *p, int64_t at, const float (&v)[8]) {
  if constexpr (F32) {
    *(f32x4_any *)((float *)p + at) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4_any *)((float *)p + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16x2_bits(v[2 * i], v[2 * i + 1]);
    __builtin_nontemporal_store(w, (u32x4_any *)((uint16_t *)p + at));
  }
}

// a lane takes 8 values of a row, the last lane of a row what is left of it
template <bool F32>
__global__ __launch_bounds__(256) void k_silu_bwd(const void *d, int64_t dld, const void *g,
                                                  int64_t gld, const void *u, int64_t uld,
                                                  const int32_t *live, int N, int I, void *dg,
                                                  int64_t dgld, void *du, int64_t duld) {
  const int64_t per_row = (I + 7) / 8, n8 = per_row * (live ? max(0, min(*live, N)) : N);
  for (int64_t c = blockIdx.x * 256ll + threadIdx.x; c < n8; c += gridDim.x * 256ll) {
    const int64_t row = c / per_row;
    const int col = (int)(c - row * per_row) * 8;
    const int64_t dat = row * dld + col, gat = row * gld + col, uat = row * uld + col;
    const int64_t dgat = row * dgld + col, duat = row * duld + col;
    if (I - col >= 8) {
      float dv[8], gv[8], uv[8];
      load8_once<F32>(d, dat, dv);
      load8_once<F32>(g, gat, gv);
      load8_once<F32>(u, uat, uv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float a, b;
        silu_grad(dv[i], gv[i], uv[i], a, b);
        gv[i] = a;
        uv[i] = b;
      }
      store8_once<F32>(dg, dgat, gv);
      store8_once<F32>(du, duat, uv);
    } else {
      for (int i = 0; i < I - col; ++i) {
        float a, b;
        silu_grad(load1<F32>(d, dat + i), load1<F32>(g, gat + i), load1<F32>(u, uat + i), a, b);
        if constexpr (F32) {
          ((float *)dg)[dgat + i] = a;
          ((float *)du)[duat + i] = b;
        } else {
          ((uint16_t *)dg)[dgat + i] = f32_to_bf16(a);
          ((uint16_t *)du)[duat + i] = f32_to_bf16(b);
        }
      }
    }
  }
}

}  // namespace

hipError_t launch_silu_backward(const void *d, int64_t dld, const void *g, int64_t gld,
                                const void *u, int64_t uld, int dtype, const int32_t *live, int N,
                                int I, void *dg, int64_t dgld, void *du, int64_t duld,
                                hipStream_t s) {
  const int64_t blocks = ((int64_t)N * ((I + 7) / 8) + 255) / 256;
  const int grid = (int)(blocks < 4096 ? blocks : 4096);
  return enqueue(dtype == AINFER_ACT_F32 ? k_silu_bwd<true> : k_silu_bwd<false>, grid, 256, s, d, dld,
                 g, gld, u, uld, live, N, I, dg, dgld, du, duld);
}

hipError_t launch_silu_rows(const void *g, int64_t gld, const void *u, int64_t uld, int in_dtype,
                            int T, int I, void *y, int64_t yld, int out_dtype, hipStream_t s) {
  const bool i32 = in_dtype == AINFER_ACT_F32, o32 = out_dtype == AINFER_ACT_F32;
  int64_t rows = T, cols = I;
  if (gld == I && uld == I && yld == I) {  // one long row
    cols *= rows;
    rows = 1;
  }
  const int64_t per = (cols + 7) / 8, n8 = per * rows;
  const int64_t blocks = (n8 + 255) / 256;
  const int grid = (int)(blocks < 4096 ? blocks : 4096);
  auto run = [&](auto kernel) {
    kernel<<<grid, 256, 0, s>>>(g, gld, u, uld, y, yld, n8, per, cols);
  };
  if (i32) run(o32 ? k_silu_rows<true, true> : k_silu_rows<true, false>);
  else run(o32 ? k_silu_rows<false, true> : k_silu_rows<false, false>);
  return hipGetLastError();
}
