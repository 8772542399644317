// moe_scored.hip - scored routing (ainfer_moe_route_scored): experts by softmax
// or sigmoid scores of given logits, a selection bias, expert groups, top-k,
// renormalised weights.  The definition is in include/ainfer_moe.h.
//
// k_route_scored: one wave per token.  The 64 lanes are cut into as many slots as there are
// groups (rounded up to a power of two); slot g holds group g, each of its
// lanes NV consecutive experts, so a group's value is a reduction over
// neighbouring lanes and a row is read in whole lines.
//
// Selection, exact in the 64-bit order of the keys:
//  1. keys in fp32: the logit itself without a bias (both scores rise with the
//     logit, so no score is computed to select), score + bias with one.  A
//     biased key is within KEY_ABS + KEY_REL * |key| of the 64-bit one.
//  2. groups are ranked against each other; where the ranking depends on a
//     difference below the keys' error, their values are redone in fp64.
//  3. t = a value that at least k lanes' maxima reach and few more: down from the
//     largest in steps of 2^20, 2^22, ... of its bits, then by halves (a compare and
//     a count of the ballot each, about 7).  Then k experts reach it, so every
//     expert of the top-k has a key >= t, less the error: about k + 5 of them,
//     compacted into LDS, one per lane.
//  4. each candidate's rank is the number of candidates above it.  Two
//     biased neighbours nearer than the error send the candidates through
//     fp64 keys (one per lane) and a second ranking.
// More than 64 candidates (a large k on full lanes) are cut by a search over all
// experts; still more (many equal keys), or fewer than k experts left (the masks),
// take k rounds of a wave-wide maximum over 64-bit keys.
//
// k_route_many: many tokens of few experts, four a wave.
//
// What bounds it.  65536 tokens of 512 experts with a bias (softmax, top-10) take 58 us:
// 36 to issue 308 vector instructions a token, meanwhile the bytes' 27 (the next token's
// logits are in flight), and the rest latency: 283 scalar instructions a token, most of
// which wait for the one before, at five waves a SIMD.  k_route_many issues vector
// instructions most of its time: 64 experts with a bias 19 us, 17 of them (148 a token),
// 60 without 9.0, 7 (62); their bytes 4.  One token takes 4.4 us, of which a launch alone
// is 2.5; 4096 tokens of 256 experts in 8 groups 7.1.
#include "moe_common.h"
#include "moe_internal.h"
#include "moe_topk.h"

// 1 / i.  A symbol that the compiler may not fold: the coefficients of exp64 then
// stay in scalar registers.  As literals (and as the library's exp has its own)
// they are held in vector registers throughout the token loop: 124 VGPRs against
// 92 at 8 experts a lane, which costs the common path its waves.
__constant__ double ainfer_scored_inv[14] = {
    0, 1.0, 1.0 / 2, 1.0 / 3, 1.0 / 4, 1.0 / 5, 1.0 / 6, 1.0 / 7,
    1.0 / 8, 1.0 / 9, 1.0 / 10, 1.0 / 11, 1.0 / 12, 1.0 / 13};

namespace {

constexpr int SR_WAVES = 4;  // tokens in flight per workgroup

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }

template <int CTRL, int RMASK>
__device__ __forceinline__ float dpp_f(float old, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL,
                                                    RMASK, 0xF, false));
}
// as unsigned keys: one instruction a step, 0 being the identity of the lanes that
// a step leaves out
__device__ __forceinline__ uint32_t wave_max_key(uint32_t v) {
  auto step = [&](auto ctrl, auto rows) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value,
                                                     decltype(rows)::value, 0xF, false));
  };
  using std::integral_constant;
  step(integral_constant<int, 0xB1>(), integral_constant<int, 0xF>());
  step(integral_constant<int, 0x4E>(), integral_constant<int, 0xF>());
  step(integral_constant<int, 0x141>(), integral_constant<int, 0xF>());
  step(integral_constant<int, 0x140>(), integral_constant<int, 0xF>());
  step(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());
  step(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_max_f(float v) {
  return key_to_float(wave_max_key(ordered_key(v)));
}
__device__ __forceinline__ float wave_sum_f(float v) {
  v += dpp_f<0xB1, 0xF>(0.f, v);
  v += dpp_f<0x4E, 0xF>(0.f, v);
  v += dpp_f<0x141, 0xF>(0.f, v);
  v += dpp_f<0x140, 0xF>(0.f, v);
  v += dpp_f<0x142, 0xA>(0.f, v);
  v += dpp_f<0x143, 0xC>(0.f, v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float readlane_f(float v, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l));
}
__device__ __forceinline__ double readlane_d(double v, int l) {
  return __builtin_bit_cast(double, readlane_u64(__builtin_bit_cast(uint64_t, v), l));
}

// partner's value at the D-th step of a reduction over aligned runs of lanes
// (D = 1, 2, 4, ... up to 32); below 4 lanes an xor, at 4 and 8 a mirror, which
// reaches another half whose lanes all hold the same value
__device__ __forceinline__ float step_f(float v, int d) {
  switch (d) {
  case 1: return dpp_f<0xB1, 0xF>(v, v);
  case 2: return dpp_f<0x4E, 0xF>(v, v);
  case 4: return dpp_f<0x141, 0xF>(v, v);
  case 8: return dpp_f<0x140, 0xF>(v, v);
  default: return __shfl_xor(v, d);
  }
}

// exp(x) in fp64 for the rare comparisons below fp32: x = n ln 2 + r, Horner's form
// of the Taylor sum to r^13 / 13! (|r| <= 0.35: 4e-18).
__device__ __forceinline__ double exp64(double x) {
  x = fmin(fmax(x, -800.0), 800.0);  // beyond: 0 and inf all the same
  const double n = rint(x * 1.4426950408889634);
  // ln 2 as its upper 32 bits and the rest
  const double r = fma(n, -0x1.a39ef35793c76p-33, fma(n, -0x1.62e42feep-1, x));
  double p = 1.0;
#pragma unroll
  for (int i = 13; i >= 1; --i) p = fma(p * r, ainfer_scored_inv[i], 1.0);
  return ldexp(p, (int)n);
}

// fp64 -> uint64 whose unsigned order is the order of the numbers
__device__ __forceinline__ uint64_t ordered_key_d(double d) {
  uint64_t u = __builtin_bit_cast(uint64_t, d);
  if ((u << 1) == 0) u = 0;
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// 1 / (1 + exp(-l)) and exp(d) (d <= 0) of the selection keys: the hardware's
// exp2 and reciprocal (1 ulp each).  Error of the sigmoid: the product l log2 e
// and its constant are off by 2^-23 |l| relative to exp, and s (1 - s) |l| <=
// 0.224, s (1 - s) <= 1/4, so 2^-23 (0.224 + 0.25) from exp, 2^-24 s from 1 +
// e, 2^-23 s from the reciprocal: below 2^-22 in all.
__device__ __forceinline__ float sigmoid_fast(float l) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l * -1.44269504088896341f));
}
__device__ __forceinline__ float exp_fast(float d) {
  return __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
}
// Bounds on a biased key's error.  Sigmoid: 2^-22, and half an ulp of the sum.
// Softmax: p = e / Z with e = exp(-d), d = max - l, off by (1.125 d + 1) 2^-23
// relative (the difference, the product with log2 e, the constant, the exp2), so
// e by 1.01 2^-23; Z by the mean of that, weighted by e (the mean d is at most
// ln 1024 = 6.9: 8.8 2^-23), and by 11 levels of additions (5.5 2^-23) and the
// reciprocal: below 17.4 2^-23 p in all, with p <= 1 / Z.
constexpr float KEY_REL = 0x1p-23f;
constexpr float SIG_ABS = 0x1p-22f, SOFT_REL = 0x1.2p-19f;
constexpr float Z_REL = 0x1.1p-19f;  // of Z and p = e / Z in fp64: (8.8 + 5.5 + 1) 2^-23
constexpr float BIAS_MOST = 1e38f;

// a logit as the definition takes it: -inf where masked, +inf the largest of its type
__device__ __forceinline__ float clean_logit(float x, float lowest) {
  return x > lowest ? fminf(x, -lowest) : neg_inf();
}
__device__ __forceinline__ float clean_bias(float b) {
  return b > neg_inf() ? fminf(fmaxf(b, -BIAS_MOST), BIAS_MOST) : neg_inf();
}

struct Row {  // one token's logits and what its keys need
  const void *base;
  int64_t ld;
  int t;
  const float *bias;
  int dtype;
  float lowest;
  float m;    // softmax: largest logit
  double z;   // softmax: sum of exp(l - m)
  __device__ __forceinline__ float logit(int e) const {
    const size_t at = (size_t)t * ld + e;
    const float x = dtype == AINFER_ACT_F32 ? ((const float *)base)[at]
                                            : bf16_to_f32(((const uint16_t *)base)[at]);
    return clean_logit(x, lowest);
  }
};

// the 64-bit key of expert e whose logit is l; masked: -inf
template <bool BIAS, bool SOFT>
__device__ double key64(const Row &r, int e, float l) {
  if constexpr (!BIAS) return (double)l;
  const float b = clean_bias(r.bias[e]);
  if (l == neg_inf() || b == neg_inf()) return -INFINITY;
  const double s =
      SOFT ? exp64((double)l - (double)r.m) / r.z : 1.0 / (1.0 + exp64(-(double)l));
  return s + (double)b;
}
// score + bias in 64 bits, also without a bias (the sum of two of a group);
// softmax without a bias: exp(l - m), the common factor left out
template <bool BIAS, bool SOFT>
__device__ double score64(const Row &r, int e, float l) {
  if constexpr (BIAS) return key64<BIAS, SOFT>(r, e, l);
  if (l == neg_inf()) return -INFINITY;
  return SOFT ? exp64((double)l - (double)r.m) : 1.0 / (1.0 + exp64(-(double)l));
}

// rank of this lane's candidate by 64-bit key, equal ones lower expert first
__device__ __forceinline__ int rank64(double d, int e, int nc) {
  int rank = 0;
  for (int j = 0; j < nc; ++j) {
    const double o = readlane_d(d, j);
    rank += (o > d || (o == d && __builtin_amdgcn_readlane(e, j) < e)) ? 1 : 0;
  }
  return rank;
}

struct Slot {  // the experts of this lane: base .. base + n - 1 of its group
  int base, n;
};

// softmax's sum in 64 bits, four terms at a time
__device__ double soft_sum64(const Row &r, const Slot &s) {
  double z = 0.0;
#pragma unroll 1
  for (int i = 0; i < s.n; i += 4) {
    float l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) l[j] = i + j < s.n ? r.logit(s.base + i + j) : neg_inf();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double e = exp64((double)fmaxf(l[j], -3.402823466e38f) - (double)r.m);
      z += l[j] != neg_inf() ? e : 0.0;
    }
  }
  return wave_sum_f64(z);
}

// value of this lane's group in 64 bits, in every lane of the group
template <bool BIAS, bool SOFT>
__device__ double group64(const Row &r, const Slot &s, int lanes, bool top2) {
  double a = -INFINITY, b = -INFINITY;  // the two largest
#pragma unroll 1
  for (int i = 0; i < s.n; ++i) {
    const int e = s.base + i;
    const float l = r.logit(e);
    const double v = top2 ? score64<BIAS, SOFT>(r, e, l) : key64<BIAS, SOFT>(r, e, l);
    if (v > a) {
      b = a;
      a = v;
    } else if (v > b) {
      b = v;
    }
  }
  for (int d = 1; d < lanes; d *= 2) {
    const double oa = __shfl_xor(a, d), ob = __shfl_xor(b, d);
    b = fmax(fmin(a, oa), fmax(b, ob));
    a = fmax(a, oa);
  }
  return top2 && b != -INFINITY ? a + b : a;
}

// rank of this lane's group by 64-bit values, equal ones lower first
__device__ int group_rank64(double v, int G, int gl, int g) {
  int rank = 0;
  for (int h = 0; h < G; ++h) {
    const double o = readlane_d(v, h << gl);
    rank += (o > v || (o == v && h < g)) ? 1 : 0;
  }
  return rank;
}

// k rounds of a wave maximum by (64-bit key, lower index): masked experts of the
// kept groups after all others.  Lane j < k returns pick j.
template <bool BIAS, bool SOFT>
__device__ int pick_rounds(const Row &r, const Slot &s, bool kept, int k, int lane) {
  uint32_t taken = 0;
  uint64_t bk = 0;  // this lane's best key left (0: none), and its expert
  int be = 0x7FFFFFFF;
  auto rescan = [&]() {
    bk = 0;
    be = 0x7FFFFFFF;
#pragma unroll 1
    for (int i = 0; i < s.n; ++i) {
      if ((taken >> i) & 1u) continue;
      const int e = s.base + i;
      // ordered_key_d(-inf) is above 0
      const uint64_t key = ordered_key_d(key64<BIAS, SOFT>(r, e, r.logit(e)));
      if (key > bk) {
        bk = key;
        be = e;
      }
    }
  };
  if (kept) rescan();
  int mine = 0;
  for (int j = 0; j < k; ++j) {
    const uint32_t hi = wave_max_u32((uint32_t)(bk >> 32));
    const uint32_t lo = wave_max_u32((uint32_t)(bk >> 32) == hi ? (uint32_t)bk : 0u);
    const bool hold = bk == (((uint64_t)hi << 32) | lo) && bk != 0;
    const uint32_t e = wave_min_u32(hold ? (uint32_t)be : 0xFFFFFFFFu);
    if (hold && (uint32_t)be == e) {
      taken |= 1u << (be - s.base);
      rescan();
    }
    if (lane == j) mine = (int)e;
  }
  return mine;
}

// A group's value gv of its two largest keys, and the errors tol of two such values:
// each of up to two keys (exp alone is off by 1.01 2^-23) and the rounding of
// their sum
template <bool BIAS, bool SOFT>
__device__ __forceinline__ void group_value(float m1, float m2, bool top2, float m, float eps_abs,
                                            float &gv, float &tol) {
  gv = m1;
  if (top2) {
    if constexpr (!BIAS) {  // the logits order the scores: the two largest give the sum
      m1 = m1 == neg_inf() ? m1 : SOFT ? exp_fast(m1 - m) : sigmoid_fast(m1);
      m2 = m2 == neg_inf() ? m2 : SOFT ? exp_fast(m2 - m) : sigmoid_fast(m2);
    }
    gv = m2 == neg_inf() ? m1 : m1 + m2;
  }
  tol = 0.0f;
  if (BIAS || top2)
    tol = 4.0f * (BIAS ? eps_abs : SIG_ABS) +
          4.0f * KEY_REL * (m2 == neg_inf() ? fabsf(gv) : fabsf(m1) + fabsf(m2));
  if (gv == neg_inf()) tol = 0.0f;
}

// A selected score relative to the largest one's, mx its logit, so that the largest
// does not vanish: exp(l - mx); sigmoid: exp(l) / (1 + exp(l)), times exp(-mx) where
// the largest logit is below 0
template <bool SOFT>
__device__ __forceinline__ float relative_score(float l, float mx) {
  if constexpr (SOFT) return exp_fast(l - mx);
  const float e = exp_fast(-fabsf(l));
  return (mx < 0.0f ? exp_fast(l - mx) : l > 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e);
}

// a lane's NV logits of one row, as loaded: whole 16- or 8-byte pieces where
// VEC allows, else one by one; what lies past the lane's experts reads as 0
template <int NV>
struct Raw {
  uint32_t v[NV];  // fp32 bits
  __device__ __forceinline__ void load(const ScoredArgs &a, int t, const Slot &s) {
    const int esz = a.dtype == AINFER_ACT_F32 ? 4 : 2;
    load(a, make_rsrc((const char *)a.logits + (size_t)t * a.ld * esz, a.G * a.per * esz), 0, esz, s);
  }
  __device__ __forceinline__ void load(const ScoredArgs &a, __amdgpu_buffer_rsrc_t r, uint32_t row,
                                       int esz, const Slot &s) {
    auto at = [&](int i) { return i < s.n ? row + (uint32_t)(s.base + i) * esz : BUF_OOB; };
    if (esz == 4) {
      if constexpr (NV >= 4) {
        if (a.vec) {
#pragma unroll
          for (int i = 0; i < NV; i += 4) {
            const u32x4 q = buf_load16(r, at(i));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = q[j];
          }
          return;
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b32(r, at(i), 0, 0);
    } else {
      if constexpr (NV >= 4) {
        if (a.vec) {
          constexpr int P = NV >= 8 ? 8 : 4;
#pragma unroll
          for (int i = 0; i < NV; i += P) {
            u32x4 q;
            if constexpr (P == 8) {
              q = buf_load16(r, at(i));
            } else {
              const u32x2 h = __builtin_bit_cast(
                  u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, at(i), 0, 0));
              q = (u32x4){h[0], h[1], 0, 0};
            }
#pragma unroll
            for (int j = 0; j < P; ++j) v[i + j] = j & 1 ? q[j / 2] & 0xFFFF0000u : q[j / 2] << 16;
          }
          return;
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
        v[i] = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at(i), 0, 0) << 16;
    }
  }
};

// The candidates of one token in a wave's LDS: key, logit, expert.
struct Cands {
  float key[64], l[64], b[64];
  int e[64];
};

template <int NV, bool BIAS, bool SOFT, bool GRP>
__global__ __launch_bounds__(64 * SR_WAVES) void k_route_scored(ScoredArgs a) {
  __shared__ __align__(16) Cands s_cand[SR_WAVES];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Cands &cand = s_cand[wave];
  const int gl = GRP ? a.gl : 6;  // log2 of a group's lanes
  const int lanes = 1 << gl;
  const int g = lane >> gl, sub = lane & (lanes - 1);
  Slot sl;
  sl.base = g * a.per + sub * a.each;
  sl.n = g < a.G ? min(max(a.per - sub * a.each, 0), a.each) : 0;
  const bool full = __ballot(sl.n == NV) == ~0ull;  // every lane has NV experts
  const int step = gridDim.x * SR_WAVES;
  int t = blockIdx.x * SR_WAVES + wave;
  if (t >= a.T) return;
  Raw<NV> raw;
  raw.load(a, t, sl);
  float b[BIAS ? NV : 1];
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {  // all in flight, without a branch
      const uint32_t v = __builtin_amdgcn_raw_buffer_load_b32(
          make_rsrc(a.bias, a.G * a.per * 4), i < sl.n ? (sl.base + i) * 4 : BUF_OOB, 0, 0);
      b[i] = __uint_as_float(v);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) b[i] = i < sl.n ? clean_bias(b[i]) : neg_inf();
  }
  Row r;
  r.base = a.logits;
  r.ld = a.ld;
  r.bias = a.bias;
  r.dtype = a.dtype;
  r.lowest = a.dtype == AINFER_ACT_F32 ? -3.402823466e38f : -3.3895313892515355e38f;
  const bool need_z = SOFT && (BIAS || !a.renorm);
  const bool need_m = SOFT && (need_z || GRP);

  for (; t < a.T; t += step) {
    r.t = t;
    float l[NV];
    bool odd = false;  // a mask, an infinity or NaN
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      l[i] = __uint_as_float(raw.v[i]);
      odd |= !(fabsf(l[i]) < -r.lowest);
    }
    if (t + step < a.T) raw.load(a, t + step, sl);  // the next token's, in flight meanwhile
    const bool masks = __ballot(odd) != 0;
    if (__builtin_expect(masks, 0)) {
      asm volatile("");  // a branch, not selects that every row pays for
#pragma unroll
      for (int i = 0; i < NV; ++i) l[i] = clean_logit(l[i], r.lowest);
    }
    if (!full) {
#pragma unroll
      for (int i = 0; i < NV; ++i) l[i] = i < sl.n ? l[i] : neg_inf();
    }

    // scores where the selection or the weights need them
    r.m = 0.0f;
    float z = 1.0f, eps_abs = SIG_ABS;
    if (need_m) {
      float m = l[0];
#pragma unroll
      for (int i = 1; i < NV; ++i) m = fmaxf(m, l[i]);
      m = wave_max_f(m);
      r.m = m == neg_inf() ? 0.0f : m;
    }
    float v[NV];  // selection keys; -inf: masked, or not there (its bias is -inf too)
    if constexpr (SOFT) {
      if (need_z) {
        float e[NV];
        float sum[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) sum[i] = e[i] = exp_fast(l[i] - r.m);  // masked: exp2(-inf) = 0
#pragma unroll
        for (int d = NV / 2; d >= 1; d /= 2)
#pragma unroll
          for (int i = 0; i < d; ++i) sum[i] += sum[i + d];
        z = wave_sum_f(sum[0]);
        if (z == 0.0f) z = 1.0f;
        if constexpr (BIAS) {
          const float rz = 1.0f / z;
          eps_abs = SOFT_REL * rz;
#pragma unroll
          for (int i = 0; i < NV; ++i) v[i] = fmaf(e[i], rz, b[i]);
        }
      }
    } else if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = sigmoid_fast(l[i]) + b[i];
    }
    if constexpr (!BIAS) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = l[i];
    } else if (masks) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = l[i] == neg_inf() ? neg_inf() : v[i];
    }

    bool have_z64 = false;
    auto z64 = [&]() {
      if (SOFT && BIAS && !have_z64) {
        r.z = soft_sum64(r, sl);
        have_z64 = true;
      }
    };

    // groups: the kept ones' lanes go on
    bool kept = GRP ? g < a.G : true;
    if constexpr (GRP) {
      const bool top2 = a.group_score == AINFER_GROUP_TOP2;
      float m1 = v[0], m2 = neg_inf();
#pragma unroll
      for (int i = 1; i < NV; ++i) {
        m2 = fmaxf(m2, fminf(m1, v[i]));
        m1 = fmaxf(m1, v[i]);
      }
      for (int d = 1; d < lanes; d *= 2) {
        const float o1 = step_f(m1, d), o2 = step_f(m2, d);
        m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
        m1 = fmaxf(m1, o1);
      }
      const bool exact = !BIAS && !top2;
      float gv, tol;
      group_value<BIAS, SOFT>(m1, m2, top2, r.m, eps_abs, gv, tol);
      const float hi_g = gv + tol, lo_g = gv - tol;
      int above = 0, near = 0;
      for (int h = 0; h < a.G; ++h) {
        const float o = readlane_f(gv, h << gl);
        above += o > hi_g ? 1 : 0;
        near += o >= lo_g ? 1 : 0;  // itself among them
      }
      kept = g < a.G && near <= a.top;
      if (__builtin_expect(__ballot(g < a.G && above < a.top && near > a.top) != 0, 0)) {
        z64();
        const double v64 = exact ? (double)gv : group64<BIAS, SOFT>(r, sl, lanes, top2);
        kept = g < a.G && group_rank64(v64, a.G, gl, g) < a.top;
      }
    }

    // a value that at least k lanes' maxima reach, and few more: down from the
    // largest in growing steps, then by halves
    float lm = v[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) lm = fmaxf(lm, v[i]);
    const uint32_t ok = kept && lm != neg_inf() ? ordered_key(lm) : 0u;
    float tf = -3.402823466e38f;
    if (__popcll(__ballot(ok != 0)) >= a.k) {
      const uint32_t most = wave_max_key(ok);
      uint32_t lo = 1, hi = most + 1;  // at least k lanes reach lo, fewer reach hi
      uint32_t down = 1u << 20;
      while (hi - lo > 1) {
        uint32_t c = lo + (hi - lo) / 2;
        if (down && most - down < hi && most - down > lo && most > down) c = most - down;
        const int n = __popcll(__ballot(ok >= c));
        if (n >= a.k) {
          lo = c;
          down = 0;
          if (n <= a.k + a.more) break;
        } else {
          hi = c;
          down *= 4;
        }
      }
      tf = key_to_float(lo);
      if constexpr (BIAS) tf -= 4.0f * eps_abs + 4.0f * KEY_REL * fabsf(tf);
    }
    if (!kept) tf = INFINITY;
    int cnt = 0, incl = 0, nc = 0;
    auto count = [&]() {
      cnt = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) cnt += v[i] >= tf ? 1 : 0;
      incl = wave_scan_incl(cnt);
      nc = __builtin_amdgcn_readlane(incl, 63);
    };
    count();
    if (__builtin_expect(nc > 64, 0)) {
      // several experts of many lanes (a large k): halve between a value that more
      // than 64 reach and one that fewer than k do
      uint32_t lo = ordered_key(-3.402823466e38f), hi = ordered_key(3.402823466e38f);
      while (hi - lo > 1) {
        const uint32_t c = lo + (hi - lo) / 2;
        const float f = key_to_float(c);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) n += __popcll(__ballot(kept && v[i] >= f));
        if (n >= a.k) lo = c;
        else hi = c;
        if (n >= a.k && n <= 48) break;
      }
      tf = key_to_float(lo);
      if constexpr (BIAS) tf -= 4.0f * eps_abs + 4.0f * KEY_REL * fabsf(tf);
      if (!kept) tf = INFINITY;
      count();
    }

    int e_mine = 0, rank = 64;
    float l_mine = neg_inf();
    if (__builtin_expect(nc >= a.k && nc <= 64, 1)) {
      int pos = incl - cnt;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (v[i] >= tf) {
          if constexpr (BIAS) {
            cand.key[pos] = v[i];
            cand.b[pos] = b[i];
          }
          cand.l[pos] = l[i];
          cand.e[pos] = sl.base + i;
          ++pos;
        }
      float *key = BIAS ? cand.key : cand.l;
      if (lane >= nc) key[lane] = neg_inf();
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const bool in = lane < nc;
      const float mine = key[lane];
      l_mine = BIAS ? cand.l[lane] : mine;
      e_mine = cand.e[lane];
      // candidates surely above this one, and not surely below it (itself among them)
      const float tol = BIAS ? 2.0f * eps_abs + 2.0f * KEY_REL * fabsf(mine) : 0.0f;
      const float hi = mine + tol, lo = mine - tol;
      int above = 0, near = 0;
      auto four = [&](const f32x4 &o) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          above += o[j] > hi ? 1 : 0;
          near += o[j] >= lo ? 1 : 0;
        }
      };
      f32x4 o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = *(const f32x4 *)&key[4 * q];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (4 * q < nc) four(o[q]);
      for (int j = 16; j < nc; j += 4) four(*(const f32x4 *)&key[j]);
      rank = above;
      if (__builtin_expect(__ballot(in && above < a.k && near - above != 1) != 0, 0)) {
        // equal keys, or biased ones nearer than their errors: in 64 bits
        if constexpr (!BIAS) {
          rank = rank64(in ? (double)mine : -INFINITY, e_mine, nc);
        } else if constexpr (!SOFT) {
          const double s = 1.0 / (1.0 + exp64(-(double)l_mine));
          rank = rank64(in ? s + (double)cand.b[lane] : -INFINITY, e_mine, nc);
        } else {
          // Z, common to all, changes a difference of keys by its error times the
          // difference of the scores: mostly the fp32 Z settles the order
          const double e = in ? exp64((double)l_mine - (double)r.m) : 0.0;
          const double be = (double)cand.b[lane];
          double p = e / (double)z, d = in ? p + be : -INFINITY;
          int sure = 0, maybe = 0;
          for (int j = 0; j < nc; ++j) {
            const double od = readlane_d(d, j), op = readlane_d(p, j);
            const double tol = fabs(op - p) * (double)Z_REL + 1e-14 * (fabs(d) + 1.0);
            sure += od - d > tol ? 1 : 0;
            maybe += od - d >= -tol ? 1 : 0;
          }
          if (__ballot(in && sure < a.k && maybe - sure != 1)) {
            z64();
            d = in ? e / r.z + be : -INFINITY;
          }
          rank = rank64(d, e_mine, nc);
        }
      }
      if (!in) rank = 64;
      __builtin_amdgcn_wave_barrier();
    } else {
      z64();
      e_mine = pick_rounds<BIAS, SOFT>(r, sl, kept, a.k, lane);
      if (lane < a.k) {
        rank = lane;
        l_mine = r.logit(e_mine);
        if (BIAS && clean_bias(r.bias[e_mine]) == neg_inf()) l_mine = neg_inf();
      }
    }

    // weights of the lanes that hold a pick
    const bool sel = rank < a.k;
    const bool live = sel && l_mine != neg_inf();
    float w;
    if (a.renorm) {
      // the selected scores over their sum
      const float mx = wave_max_f(live ? l_mine : neg_inf());
      const float s = live ? relative_score<SOFT>(l_mine, mx) : 0.0f;
      const float sum = wave_sum_f(s);
      w = sum > 0.0f ? s * __builtin_amdgcn_rcpf(sum) * a.scale : 0.0f;
    } else if constexpr (SOFT) {
      w = live ? exp_fast(l_mine - r.m) * __builtin_amdgcn_rcpf(z) * a.scale : 0.0f;
    } else {
      w = live ? sigmoid_fast(l_mine) * a.scale : 0.0f;
    }
    if (sel) {
      a.idx[(size_t)t * a.k + rank] = e_mine;
      a.w[(size_t)t * a.k + rank] = w;
    }
  }
}

// ---- many tokens of few experts -------------------------------------------------
//
// Four tokens a wave, 16 lanes each (the slots of the groups within them), since
// what a wave does for a token above costs the same however few its experts are.
// k rounds of the largest key left of 16 lanes, ties to the lowest lane and there to
// the lowest expert; lanes hold experts in ascending order.  With a bias one round
// more: where two picks are nearer than the keys' errors, they are ranked by 64-bit
// keys, and where the last and the next are, the rounds are run again on those.

template <class F>
__device__ __forceinline__ float reduce16(float v, F f) {
  v = f(v, dpp_f<0xB1, 0xF>(v, v));
  v = f(v, dpp_f<0x4E, 0xF>(v, v));
  v = f(v, dpp_f<0x141, 0xF>(v, v));
  return f(v, dpp_f<0x140, 0xF>(v, v));
}
__device__ __forceinline__ float max16(float v) {
  return reduce16(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float sum16(float v) {
  return reduce16(v, [](float x, float y) { return x + y; });
}
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
}
__device__ __forceinline__ uint64_t max16(uint64_t v) {
  v = max_u64(v, dpp_u64<0xB1>(v));
  v = max_u64(v, dpp_u64<0x4E>(v));
  v = max_u64(v, dpp_u64<0x141>(v));
  return max_u64(v, dpp_u64<0x140>(v));
}

struct Pick {
  int e;
  float l;
};
constexpr int MP_K = 16;  // picks of a token: one a lane

template <int NV, bool BIAS, bool SOFT, bool GRP>
__global__ __launch_bounds__(64 * SR_WAVES) void k_route_many(ScoredArgs a) {
  __shared__ Pick s_pick[SR_WAVES][4][MP_K];
  const int lane = threadIdx.x & 63, lane16 = lane & 15, seg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = (blockIdx.x * SR_WAVES + wave) * 4, t = t0 + seg;
  if (t0 >= a.T) return;
  const int gl = GRP ? a.gl : 4, lanes = 1 << gl;
  const int g = lane16 >> gl, sub = lane16 & (lanes - 1);
  Slot sl;
  sl.base = g * a.per + sub * NV;
  sl.n = g < a.G && t < a.T ? min(max(a.per - sub * NV, 0), NV) : 0;
  const int esz = a.dtype == AINFER_ACT_F32 ? 4 : 2;
  Raw<NV> raw;
  raw.load(a, make_rsrc((const char *)a.logits + (size_t)t0 * a.ld * esz, 0x7FFFFFFFu),
           (uint32_t)(seg * a.ld) * esz, esz, sl);
  float b[BIAS ? NV : 1];
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      b[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
          make_rsrc(a.bias, a.G * a.per * 4), i < sl.n ? (sl.base + i) * 4 : BUF_OOB, 0, 0));
#pragma unroll
    for (int i = 0; i < NV; ++i) b[i] = clean_bias(b[i]);
  }
  Row r;
  r.base = a.logits;
  r.ld = a.ld;
  r.t = t;
  r.bias = a.bias;
  r.dtype = a.dtype;
  r.lowest = a.dtype == AINFER_ACT_F32 ? -3.402823466e38f : -3.3895313892515355e38f;
  r.m = 0.0f;
  float l[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    l[i] = i < sl.n ? clean_logit(__uint_as_float(raw.v[i]), r.lowest) : neg_inf();

  const bool need_z = SOFT && (BIAS || !a.renorm);
  float z = 1.0f, eps_abs = SIG_ABS;
  if (SOFT && (need_z || GRP)) {
    float m = l[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, l[i]);
    m = max16(m);
    r.m = m == neg_inf() ? 0.0f : m;
  }
  float v[NV];  // selection keys; -inf: masked
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = l[i];
  if constexpr (SOFT) {
    if (need_z) {
      float e[NV], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) sum += e[i] = exp_fast(l[i] - r.m);
      z = sum16(sum);
      if (z == 0.0f) z = 1.0f;
      if constexpr (BIAS) {
        const float rz = 1.0f / z;
        eps_abs = SOFT_REL * rz;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = l[i] == neg_inf() ? l[i] : fmaf(e[i], rz, b[i]);
      }
    }
  } else if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = l[i] == neg_inf() ? l[i] : sigmoid_fast(l[i]) + b[i];
  }
  bool have_z64 = false;
  auto z64 = [&]() {
    if (SOFT && BIAS && !have_z64) {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        s += l[i] != neg_inf() ? exp64((double)l[i] - (double)r.m) : 0.0;
      for (int d = 1; d < 16; d *= 2) s += __shfl_xor(s, d);
      r.z = s;
      have_z64 = true;
    }
  };

  bool kept = sl.n > 0;
  if constexpr (GRP) {
    const bool top2 = a.group_score == AINFER_GROUP_TOP2;
    float m1 = v[0], m2 = neg_inf();
#pragma unroll
    for (int i = 1; i < NV; ++i) {
      m2 = fmaxf(m2, fminf(m1, v[i]));
      m1 = fmaxf(m1, v[i]);
    }
    for (int d = 1; d < lanes; d *= 2) {
      const float o1 = step_f(m1, d), o2 = step_f(m2, d);
      m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
      m1 = fmaxf(m1, o1);
    }
    const bool exact = !BIAS && !top2;
    float gv, tol;
    group_value<BIAS, SOFT>(m1, m2, top2, r.m, eps_abs, gv, tol);
    const float hi_g = gv + tol, lo_g = gv - tol;
    const int slots = 16 >> gl;
    int above = 0, near = 1;
    for (int d = 1; d < slots; ++d) {
      const int h = (g + d) & (slots - 1);
      const float o = __shfl(gv, (lane & 48) | (h << gl));
      above += h < a.G && o > hi_g ? 1 : 0;
      near += h < a.G && o >= lo_g ? 1 : 0;
    }
    bool in = near <= a.top;
    if (__builtin_expect(__ballot(g < a.G && above < a.top && near > a.top) != 0, 0)) {
      z64();
      const double v64 = exact ? (double)gv : group64<BIAS, SOFT>(r, sl, lanes, top2);
      int rank = 0;
      for (int h = 0; h < a.G; ++h) {
        const double o = __shfl(v64, (lane & 48) | (h << gl));
        rank += o > v64 || (o == v64 && h < g) ? 1 : 0;
      }
      in = rank < a.top;
    }
    kept = kept && in;
  }

  // rounds: u = ordered keys (0: not there), taken ones cleared.  Bit lane of
  // `lower` stands for the lower lanes of the same token.
  const uint64_t lower = ((1ull << lane16) - 1) << (seg * 16);
  Pick *pick = s_pick[wave][seg];
  const int rounds = a.k + (BIAS ? 1 : 0);
  bool near_in = false, near_out = false;  // two picks, or the last and the next one
  auto select = [&](auto(&u)[NV], auto masked, auto &&see) {
    using U = typename std::remove_reference<decltype(u[0])>::type;
    for (int j = 0; j < rounds; ++j) {
      U best = u[0];
#pragma unroll
      for (int i = 1; i < NV; ++i) best = u[i] > best ? u[i] : best;
      const U top = max16(best);
      see(j, top);
      const bool win = best == top && (__ballot(best == top) & lower) == 0;
      int e = 0;
      float le = neg_inf();
      bool found = !win;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool hit = !found && u[i] == top;
        e = hit ? i : e;
        if (BIAS) le = hit ? l[i] : le;
        u[i] = hit ? (U)0 : u[i];
        found |= hit;
      }
      if (win && j < a.k) {
        if (BIAS) le = top == (U)masked ? neg_inf() : le;
        else le = key_to_float((uint32_t)top);
        pick[j] = Pick{sl.base + e, le};
      }
    }
  };
  {
    uint32_t u[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) u[i] = kept && i < sl.n ? ordered_key(v[i]) : 0u;
    float last = INFINITY;
    select(u, ordered_key(neg_inf()), [&](int j, uint32_t top) {
      if constexpr (BIAS) {
        const float f = key_to_float(top);  // NaN: none left
        const bool near = f != neg_inf() && last - f <= 4.0f * eps_abs + 4.0f * KEY_REL * fabsf(f);
        near_in |= near && j < a.k;
        near_out |= near && j == a.k;
        last = f;
      }
    });
    if constexpr (BIAS) {
      if (__builtin_expect(__ballot(near_out) != 0, 0)) {
        near_in = false;
        z64();
        uint64_t w[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
          w[i] = kept && i < sl.n ? ordered_key_d(key64<BIAS, SOFT>(r, sl.base + i, l[i])) : 0ull;
        select(w, ordered_key_d(-INFINITY), [](int, uint64_t) {});
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const bool sel = lane16 < a.k && t < a.T;
  const Pick mine = pick[lane16 < a.k ? lane16 : 0];
  int pos = lane16;
  if (BIAS && __builtin_expect(__ballot(near_in) != 0, 0)) {
    z64();
    const double d = sel ? key64<BIAS, SOFT>(r, mine.e, mine.l) : -INFINITY;
    pos = 0;
    for (int j = 0; j < a.k; ++j) {
      const double o = __shfl(d, (lane & 48) | j);
      const int oe = __shfl(mine.e, (lane & 48) | j);
      pos += o > d || (o == d && oe < mine.e) ? 1 : 0;
    }
  }
  const bool live = sel && mine.l != neg_inf();
  float w;
  if (a.renorm) {
    const float mx = max16(live ? mine.l : neg_inf());
    const float s = live ? relative_score<SOFT>(mine.l, mx) : 0.0f;
    const float sum = sum16(s);
    w = sum > 0.0f ? s * __builtin_amdgcn_rcpf(sum) * a.scale : 0.0f;
  } else if constexpr (SOFT) {
    w = live ? exp_fast(mine.l - r.m) * __builtin_amdgcn_rcpf(z) * a.scale : 0.0f;
  } else {
    w = live ? sigmoid_fast(mine.l) * a.scale : 0.0f;
  }
  if (sel) {
    a.idx[(size_t)t * a.k + pos] = mine.e;
    a.w[(size_t)t * a.k + pos] = w;
  }
}

template <int NV>
void launch_many(const ScoredArgs &a, bool soft, hipStream_t s) {
  const dim3 grid((a.T + SR_WAVES * 4 - 1) / (SR_WAVES * 4)), b(64 * SR_WAVES);
  auto run = [&](auto kernel) { kernel<<<grid, b, 0, s>>>(a); };
  if (a.G > 1) {
    if (a.bias) run(soft ? k_route_many<NV, true, true, true> : k_route_many<NV, true, false, true>);
    else run(soft ? k_route_many<NV, false, true, true> : k_route_many<NV, false, false, true>);
  } else {
    if (a.bias) run(soft ? k_route_many<NV, true, true, false> : k_route_many<NV, true, false, false>);
    else run(soft ? k_route_many<NV, false, true, false> : k_route_many<NV, false, false, false>);
  }
}

template <int NV, bool GRP>
void launch_grp(const ScoredArgs &a, int grid, bool soft, hipStream_t s) {
  const dim3 b(64 * SR_WAVES);
  if (a.bias) {
    if (soft) k_route_scored<NV, true, true, GRP><<<grid, b, 0, s>>>(a);
    else k_route_scored<NV, true, false, GRP><<<grid, b, 0, s>>>(a);
  } else {
    if (soft) k_route_scored<NV, false, true, GRP><<<grid, b, 0, s>>>(a);
    else k_route_scored<NV, false, false, GRP><<<grid, b, 0, s>>>(a);
  }
}
template <int NV>
void launch_nv(const ScoredArgs &a, int grid, bool soft, hipStream_t s) {
  if (a.G > 1) launch_grp<NV, true>(a, grid, soft, s);
  else launch_grp<NV, false>(a, grid, soft, s);
}

// k_route_many from this many tokens on, and while the rounds over a lane's experts
// are fewer than MANY_WORK.  us by a wave a token and by 4: T 4096 without a bias 60
// experts 4.4 and 3.2, 40 in 8 groups 6.0 and 4.6, 128 4.9 and 4.85 (T 1024 3.6 and 4.6),
// T 65536 28.6 and 8.9, 48 and 14.8, 34.9 and 17.6; with a bias, where a wave in a
// hundred has to rank 64-bit keys, T 4096 64 experts 4.9 and 6.4, T 16384 10.8 and 8.4,
// T 65536 32.9 and 19.2, 128 experts in 8 groups 51.6 and 32.8, 16 picks of 128 41.0 and
// 45.5.
constexpr int MANY_T = 4096, MANY_T_BIAS = 16384, MANY_WORK = 64;

}  // namespace

hipError_t launch_route_scored(const ainfer_moe_routing &r, const void *logits, int dtype,
                               int64_t ld, const float *bias, int T, int32_t *idx, float *w,
                               hipStream_t s) {
  ScoredArgs a;
  a.logits = logits;
  a.bias = bias;
  a.idx = idx;
  a.w = w;
  a.ld = ld;
  a.dtype = dtype;
  a.T = T;
  a.k = r.top_k;
  a.G = r.n_groups;
  a.top = r.top_groups;
  a.per = r.n_experts / r.n_groups;
  a.group_score = r.group_score;
  a.renorm = r.renormalize;
  a.scale = r.scale;
  // whole pieces of 4 (8 bf16 from 8 experts a lane on) experts, dwords aligned
  auto vec = [&](int need) {
    if (dtype == AINFER_ACT_F32) return a.per % 4 == 0;
    return a.per % (need > 4 ? 8 : 4) == 0 && (uintptr_t)logits % 4 == 0 && ld % 2 == 0;
  };
  int slots = 1;
  while (slots < a.G) slots *= 2;
  const bool soft = r.score == AINFER_SCORE_SOFTMAX;
  if (slots <= 16 && a.k <= MP_K && T >= (bias ? MANY_T_BIAS : MANY_T) &&
      (3 * ld + r.n_experts) * 4 < INT32_MAX) {
    for (a.gl = 0; (slots << a.gl) < 16;) ++a.gl;
    const int need = (a.per + (1 << a.gl) - 1) >> a.gl;
    a.vec = vec(need);
    if (need <= 8 && a.k * need <= MANY_WORK) {
      if (need <= 1) launch_many<1>(a, soft, s);
      else if (need <= 2) launch_many<2>(a, soft, s);
      else if (need <= 4) launch_many<4>(a, soft, s);
      else launch_many<8>(a, soft, s);
      return hipGetLastError();
    }
  }
  a.gl = 0;
  while ((slots << a.gl) < 64) ++a.gl;
  a.more = a.k <= 16 ? 3 : 0;
  const int lanes = 1 << a.gl, need = (a.per + lanes - 1) / lanes;
  a.vec = vec(need);
  // experts a lane, of the NV it has room for: shared evenly, so that the maxima of many
  // lanes bound the top-k (one group of 291 in lanes of 32: 10 maxima, 16 us; of 19: 8)
  const int piece = !a.vec || need <= 4 ? 1 : dtype == AINFER_ACT_F32 ? 4 : 8;
  a.each = need <= 4 ? (need > 2 ? 4 : need) : (need + piece - 1) / piece * piece;
  const int blocks = (T + SR_WAVES - 1) / SR_WAVES;
  // a wave keeps the bias over its tokens; without one a workgroup per 4 tokens.  us at
  // T 65536, grids of 2048 and 16384: 512 experts with a bias 64 and 93, without
  // 52 and 45 (bf16, not renormalised 70 and 53), 64 experts 38 and 31.  With 8 experts a
  // lane 1280 are resident at once (about 90 registers): 512 experts softmax 58.2 (2048
  // 60.3), sigmoid 50.2 (53.2)
  const int most = !bias ? 16384 : need > 4 && need <= 8 ? 1280 : 2048;
  const int grid = blocks < most ? blocks : most;
  if (need <= 1) launch_nv<1>(a, grid, soft, s);
  else if (need <= 2) launch_nv<2>(a, grid, soft, s);
  else if (need <= 4) launch_nv<4>(a, grid, soft, s);
  else if (need <= 8) launch_nv<8>(a, grid, soft, s);
  else if (need <= 16) launch_nv<16>(a, grid, soft, s);
  else if (a.G > 1) launch_grp<32, true>(a, grid, soft, s);
  else return hipErrorInvalidValue;  // more than 1024 experts
  return hipGetLastError();
}
