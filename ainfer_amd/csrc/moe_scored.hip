// moe_scored.hip - scored routing (ainfer_moe_route_scored): experts by softmax
// or sigmoid scores of given logits, a selection bias, expert groups, top-k,
// renormalised weights.  The definition is in include/ainfer_moe.h.
//
// One wave per token.  The 64 lanes are cut into as many slots as there are
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
//  3. t = a value that k lanes' maxima reach (a search over the bits of the
//     maxima: one compare and a count of the ballot per bit).  Then k experts
//     reach it, so every expert of the top-k has a key >= t, less the error:
//     about k + 1 of them, compacted into LDS, one per lane.
//  4. each candidate's rank is the number of candidates above it.  Two
//     biased neighbours nearer than the error send the candidates through
//     fp64 keys (one per lane) and a second ranking.
// More than 64 candidates (many equal keys), or fewer than k experts left (the
// masks), take k rounds of a wave-wide maximum over 64-bit keys.
#include "moe_common.h"
#include "moe_internal.h"
#include "moe_topk.h"

namespace {

constexpr int SR_WAVES = 4;  // tokens in flight per workgroup

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }

template <int CTRL, int RMASK>
__device__ __forceinline__ float dpp_f(float old, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL,
                                                    RMASK, 0xF, false));
}
__device__ __forceinline__ float wave_max_f(float v) {
  v = fmaxf(v, dpp_f<0xB1, 0xF>(v, v));
  v = fmaxf(v, dpp_f<0x4E, 0xF>(v, v));
  v = fmaxf(v, dpp_f<0x141, 0xF>(v, v));
  v = fmaxf(v, dpp_f<0x140, 0xF>(v, v));
  v = fmaxf(v, dpp_f<0x142, 0xA>(v, v));
  v = fmaxf(v, dpp_f<0x143, 0xC>(v, v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
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
// Softmax: p = e / Z, e = exp(l - max) off by 2^-23 |l - max| 1.5 + 2^-23, and
// e |l - max| <= 0.37; Z is a sum of at most 1024 such terms, relative error below
// 2^-23 1.5 (mean |l - max| by weight, below 10) + 38 2^-24 (32 in a lane, 6
// across): below 2^-18 p in all, with p <= 1 / Z.
constexpr float KEY_REL = 0x1p-23f;
constexpr float SIG_ABS = 0x1p-22f, SOFT_REL = 0x1p-18f;
constexpr float BIAS_MOST = 1e38f;

// a logit as the definition takes it: -inf where masked, +inf the largest
__device__ __forceinline__ float clean_logit(float x, float lowest) {
  return x > lowest ? fminf(x, 3.402823466e38f) : neg_inf();
}
__device__ __forceinline__ float clean_bias(float b) {
  return b > neg_inf() ? fminf(fmaxf(b, -BIAS_MOST), BIAS_MOST) : neg_inf();
}

struct Row {  // one token's logits and what its keys need
  const void *p;
  const float *bias;
  int dtype;
  float lowest;
  float m;    // softmax: largest logit
  double z;   // softmax: sum of exp(l - m)
  __device__ __forceinline__ float logit(int e) const {
    const float x = dtype == AINFER_ACT_F32 ? ((const float *)p)[e]
                                            : bf16_to_f32(((const uint16_t *)p)[e]);
    return clean_logit(x, lowest);
  }
};

// the 64-bit key of expert e whose logit is l; masked: -inf
template <bool BIAS, bool SOFT>
__device__ double key64(const Row &r, int e, float l) {
  if constexpr (!BIAS) return (double)l;
  const float b = clean_bias(r.bias[e]);
  if (l == neg_inf() || b == neg_inf()) return -INFINITY;
  const double s = SOFT ? exp((double)l - (double)r.m) / r.z : 1.0 / (1.0 + exp(-(double)l));
  return s + (double)b;
}
// score + bias in 64 bits, also without a bias (the sum of two of a group);
// softmax without a bias: exp(l - m), the common factor left out
template <bool BIAS, bool SOFT>
__device__ double score64(const Row &r, int e, float l) {
  if constexpr (BIAS) return key64<BIAS, SOFT>(r, e, l);
  if (l == neg_inf()) return -INFINITY;
  return SOFT ? exp((double)l - (double)r.m) : 1.0 / (1.0 + exp(-(double)l));
}

struct Slot {  // the experts of this lane: base .. base + n - 1 of its group
  int base, n;
};

// softmax's sum in 64 bits
__device__ double soft_sum64(const Row &r, const Slot &s) {
  double z = 0.0;
#pragma unroll 1
  for (int i = 0; i < s.n; ++i) {
    const float l = r.logit(s.base + i);
    if (l != neg_inf()) z += exp((double)l - (double)r.m);
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

struct Cand {  // one candidate in LDS: ordered key and ~expert (one 64-bit
  uint64_t c;  // order: key up, then lower expert), and its logit
  float l;
  uint32_t e;
};

template <int NV, bool BIAS, bool SOFT>
__global__ __launch_bounds__(64 * SR_WAVES) void k_route_scored(ScoredArgs a) {
  __shared__ Cand s_cand[SR_WAVES][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Cand *cand = s_cand[wave];
  const int lanes = 1 << a.gl;  // lanes of a group's slot
  const int g = lane >> a.gl, sub = lane & (lanes - 1);
  Slot sl;
  sl.base = g * a.per + sub * NV;
  sl.n = g < a.G ? min(max(a.per - sub * NV, 0), NV) : 0;
  const bool f32 = a.dtype == AINFER_ACT_F32;
  const size_t esz = f32 ? 4 : 2;
  float b[BIAS ? NV : 1];
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < NV; ++i) b[i] = i < sl.n ? clean_bias(a.bias[sl.base + i]) : neg_inf();
  }
  Row r;
  r.bias = a.bias;
  r.dtype = a.dtype;
  r.lowest = f32 ? -3.402823466e38f : -3.3895313892515355e38f;
  const bool need_z = SOFT && (BIAS || !a.renorm);
  const bool need_m = SOFT && (need_z || a.G > 1);

  for (int t = blockIdx.x * SR_WAVES + wave; t < a.T; t += gridDim.x * SR_WAVES) {
    r.p = (const char *)a.logits + (size_t)t * a.ld * esz;
    float l[NV];
    {
#pragma unroll
      for (int i = 0; i < NV; ++i) l[i] = neg_inf();
      bool done = false;
      if constexpr (NV >= 4) {
        if (f32 && a.vec) {  // whole 16-byte pieces: per is a multiple of 4
          const float *p = (const float *)r.p + sl.base;
#pragma unroll
          for (int i = 0; i < NV; i += 4)
            if (i < sl.n) {
              const f32x4 v = *(const f32x4 *)(p + i);
#pragma unroll
              for (int q = 0; q < 4; ++q) l[i + q] = v[q];
            }
          done = true;
        }
      }
      if constexpr (NV >= 8) {
        if (!f32 && a.vec) {  // per is a multiple of 8
          const uint16_t *p = (const uint16_t *)r.p + sl.base;
#pragma unroll
          for (int i = 0; i < NV; i += 8)
            if (i < sl.n) {
              const u32x4 v = *(const u32x4 *)(p + i);
#pragma unroll
              for (int q = 0; q < 8; ++q)
                l[i + q] = __uint_as_float(q & 1 ? v[q / 2] & 0xFFFF0000u : v[q / 2] << 16);
            }
          done = true;
        }
      }
      if (!done) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i < sl.n)
            l[i] = f32 ? ((const float *)r.p)[sl.base + i]
                       : bf16_to_f32(((const uint16_t *)r.p)[sl.base + i]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) l[i] = clean_logit(l[i], r.lowest);
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
    float v[NV];  // selection keys
    if constexpr (SOFT) {
      if (need_z) {
        float e[NV];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          e[i] = exp_fast(l[i] - r.m);  // masked: exp2(-inf) = 0
          sum += e[i];
        }
        z = wave_sum_f(sum);
        if (z == 0.0f) z = 1.0f;
        if constexpr (BIAS) {
          const float rz = 1.0f / z;
          eps_abs = SOFT_REL * rz;
#pragma unroll
          for (int i = 0; i < NV; ++i) v[i] = l[i] == neg_inf() ? neg_inf() : fmaf(e[i], rz, b[i]);
        }
      }
    } else if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = l[i] == neg_inf() ? neg_inf() : sigmoid_fast(l[i]) + b[i];
    }
    if constexpr (!BIAS) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = l[i];
    }

    bool have_z64 = false;
    auto z64 = [&]() {
      if (SOFT && BIAS && !have_z64) {
        r.z = soft_sum64(r, sl);
        have_z64 = true;
      }
    };

    // groups: the kept ones' lanes go on
    bool kept = g < a.G;
    if (a.G > 1) {
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
      float gv = m1, eps = 0.0f;
      if (top2) {
        if constexpr (!BIAS) {  // the logits order the scores: the two largest give the sum
          m1 = m1 == neg_inf() ? m1 : SOFT ? exp_fast(m1 - r.m) : sigmoid_fast(m1);
          m2 = m2 == neg_inf() ? m2 : SOFT ? exp_fast(m2 - r.m) : sigmoid_fast(m2);
        }
        gv = m2 == neg_inf() ? m1 : m1 + m2;
        // exp alone is off by 2^-22.4 (0.37 1.5 2^-23 + 2^-23)
        eps = 2.0f * (BIAS ? eps_abs : SIG_ABS) + KEY_REL * (fabsf(m1) + fabsf(m2));
      } else if constexpr (BIAS) {
        eps = eps_abs + KEY_REL * fabsf(m1);
      }
      if (gv == neg_inf()) eps = 0.0f;
      int rank = 0, above = 0, near = 0;
      for (int h = 0; h < a.G; ++h) {
        const float o = readlane_f(gv, h << a.gl), oe = readlane_f(eps, h << a.gl);
        const float d = o - gv, e = oe + eps;  // both -inf: d is NaN, equal
        rank += (o > gv || (o == gv && h < g)) ? 1 : 0;
        above += d > e ? 1 : 0;
        near += d < -e ? 0 : 1;  // itself among them
      }
      const bool exact = !BIAS && !top2;
      if (!exact && __ballot(g < a.G && above < a.top && near > a.top)) {
        z64();
        rank = group_rank64(group64<BIAS, SOFT>(r, sl, lanes, top2), a.G, a.gl, g);
      }
      kept = g < a.G && rank < a.top;
    }

    // a value that k lanes' maxima reach
    float lm = v[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) lm = fmaxf(lm, v[i]);
    const uint32_t ok = kept && lm != neg_inf() ? ordered_key(lm) : 0u;
    float tf = -3.402823466e38f;
    if (__popcll(__ballot(ok != 0)) >= a.k) {
      uint32_t tk = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = tk | (1u << bit);
        const int n = __popcll(__ballot(ok >= c));
        if (n >= a.k) tk = c;
        if (n == a.k) break;
      }
      tf = key_to_float(tk);
      if constexpr (BIAS) tf -= 4.0f * eps_abs + 4.0f * KEY_REL * fabsf(tf);
    }
    if (!kept) tf = INFINITY;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) cnt += v[i] >= tf ? 1 : 0;
    const int incl = wave_scan_incl(cnt);
    const int nc = __builtin_amdgcn_readlane(incl, 63);

    int e_mine = 0, rank = 64;
    float l_mine = neg_inf();
    if (nc >= a.k && nc <= 64) {
      int pos = incl - cnt;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (v[i] >= tf) {
          Cand c;
          c.c = ((uint64_t)ordered_key(v[i]) << 32) | (uint32_t)~(uint32_t)(sl.base + i);
          c.l = l[i];
          c.e = sl.base + i;
          cand[pos++] = c;
        }
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const bool in = lane < nc;
      const uint64_t mine = in ? cand[lane].c : 0;
      if (in) {
        e_mine = (int)cand[lane].e;
        l_mine = cand[lane].l;
      }
      rank = 0;
      for (int j = 0; j < nc; ++j) rank += cand[j].c > mine ? 1 : 0;
      if constexpr (BIAS) {
        // the candidates in order: neighbours nearer than their errors?
        const float key = key_to_float((uint32_t)(mine >> 32));
        const int src = __builtin_amdgcn_ds_permute(4 * (in ? rank : lane), __float_as_int(key));
        const float ks = __int_as_float(src);
        const float nx = __shfl_down(ks, 1);
        const bool near = lane + 1 < nc && lane < a.k &&
                          !(ks - nx > 2.0f * eps_abs + 2.0f * KEY_REL * fmaxf(fabsf(ks), fabsf(nx)));
        if (__ballot(near)) {
          z64();
          const double d = in ? key64<BIAS, SOFT>(r, e_mine, l_mine) : -INFINITY;
          rank = 0;
          for (int j = 0; j < nc; ++j) {
            const double o = readlane_d(d, j);
            rank += (o > d || (o == d && __builtin_amdgcn_readlane(e_mine, j) < e_mine)) ? 1 : 0;
          }
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
      // the selected scores over their sum, scaled so that the largest does not
      // vanish: exp(l - max), or exp(l - c) / (1 + exp(l)) with c the largest
      // logit where that is negative
      const float mx = wave_max_f(live ? l_mine : neg_inf());
      float s = 0.0f;
      if (live) {
        if constexpr (SOFT) {
          s = expf(l_mine - mx);
        } else {
          s = l_mine > 0.0f ? 1.0f / (1.0f + expf(-l_mine))
                            : expf(l_mine - fminf(mx, 0.0f)) / (1.0f + expf(l_mine));
        }
      }
      const float sum = wave_sum_f(s);
      w = sum > 0.0f ? s / sum * a.scale : 0.0f;
    } else if (!live) {
      w = 0.0f;
    } else if constexpr (SOFT) {
      w = expf(l_mine - r.m) / z * a.scale;
    } else {
      w = 1.0f / (1.0f + expf(-l_mine)) * a.scale;
    }
    if (sel) {
      a.idx[(size_t)t * a.k + rank] = e_mine;
      a.w[(size_t)t * a.k + rank] = w;
    }
  }
}

template <int NV>
void launch_nv(const ScoredArgs &a, int grid, bool soft, hipStream_t s) {
  const dim3 b(64 * SR_WAVES);
  if (a.bias) {
    if (soft)
      k_route_scored<NV, true, true><<<grid, b, 0, s>>>(a);
    else
      k_route_scored<NV, true, false><<<grid, b, 0, s>>>(a);
  } else {
    if (soft)
      k_route_scored<NV, false, true><<<grid, b, 0, s>>>(a);
    else
      k_route_scored<NV, false, false><<<grid, b, 0, s>>>(a);
  }
}

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
  int slots = 1;
  while (slots < a.G) slots *= 2;
  a.gl = 0;
  while ((slots << a.gl) < 64) ++a.gl;
  const int lanes = 1 << a.gl, need = (a.per + lanes - 1) / lanes;
  const int esz = dtype == AINFER_ACT_F32 ? 4 : 2, piece = 16 / esz;
  a.vec = a.per % piece == 0 && (uintptr_t)logits % 16 == 0 && (ld * esz) % 16 == 0;
  const int blocks = (T + SR_WAVES - 1) / SR_WAVES;
  const int grid = blocks < SR_MAX_GRID ? blocks : SR_MAX_GRID;
  const bool soft = r.score == AINFER_SCORE_SOFTMAX;
  if (need <= 1) launch_nv<1>(a, grid, soft, s);
  else if (need <= 2) launch_nv<2>(a, grid, soft, s);
  else if (need <= 4) launch_nv<4>(a, grid, soft, s);
  else if (need <= 8) launch_nv<8>(a, grid, soft, s);
  else if (need <= 16) launch_nv<16>(a, grid, soft, s);
  else launch_nv<32>(a, grid, soft, s);
  return hipGetLastError();
}
