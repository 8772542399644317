// moe_api.hip - the C ABI of include/ainfer_moe.h: validation, workspace
// layout and the stage sequence router -> top-k -> dispatch -> gate/up ->
// down -> combine.  Host code; every device buffer comes from the caller.
#include <string.h>

#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <vector>

#include "moe_common.h"
#include "moe_internal.h"

namespace {

// ---- profiling: one event per stage boundary, per call ---------------------
constexpr int NSTAGE = AINFER_MOE_N_STAGES;
constexpr int PROF_SLOTS = 64;
struct Prof {
  bool on = false;
  bool created = false;
  hipEvent_t ev[PROF_SLOTS][NSTAGE + 1];
  bool used[PROF_SLOTS][NSTAGE + 1];
  int slot = 0, calls = 0;
  double sum_us[NSTAGE];
  int cnt[NSTAGE];
  // the decode gate/up kernel's own start and end (hipExtLaunchKernel events,
  // stamped by the dispatch: no barrier packets of their own)
  hipEvent_t kev[PROF_SLOTS][2];
  bool kused[PROF_SLOTS];
  double ksum_us;
  int kcnt;
} g_prof;

void prof_flush_slot(int s) {
  // stage i spans the last recorded event before it to its own end event
  int prev = -1;
  for (int i = 0; i <= NSTAGE; ++i) {
    if (!g_prof.used[s][i]) continue;
    if (prev >= 0) {
      (void)hipEventSynchronize(g_prof.ev[s][i]);
      float ms = 0.f;
      if (hipEventElapsedTime(&ms, g_prof.ev[s][prev], g_prof.ev[s][i]) == hipSuccess) {
        g_prof.sum_us[i - 1] += ms * 1000.0;
        g_prof.cnt[i - 1] += 1;
      }
    }
    prev = i;
    g_prof.used[s][i] = false;
  }
  if (g_prof.kused[s]) {
    float ms = 0.f;
    if (hipEventSynchronize(g_prof.kev[s][1]) == hipSuccess &&
        hipEventElapsedTime(&ms, g_prof.kev[s][0], g_prof.kev[s][1]) == hipSuccess) {
      g_prof.ksum_us += ms * 1000.0;
      g_prof.kcnt += 1;
    }
    g_prof.kused[s] = false;
  }
}

struct ProfCall {
  int s = -1;
  hipStream_t st;
  explicit ProfCall(hipStream_t stream) : st(stream) {
    if (!g_prof.on) return;
    s = g_prof.slot;
    g_prof.slot = (g_prof.slot + 1) % PROF_SLOTS;
    prof_flush_slot(s);  // reuse: collect the slot's previous call first
    g_prof.calls++;
  }
  // mark the end of stage `stage` (index = stage + 1); the call's first
  // mark is the start event
  void start() {
    if (s >= 0) rec(0);
  }
  void end(int stage) {
    if (s >= 0) rec(stage + 1);
  }
  void rec(int i) {
    (void)hipEventRecord(g_prof.ev[s][i], st);
    g_prof.used[s][i] = true;
  }
  // the next gate/up expert launch records its own start and end
  void kernel_events() {
    if (s < 0) return;
    set_expert_launch_events(g_prof.kev[s][0], g_prof.kev[s][1]);
    g_prof.kused[s] = true;
  }
};

struct Layout {
  size_t w8_xq, w8_xs, w8_act, w8_acts, w8_aq, w8_as, w8_aqs, w8_ass, w8_o;
  size_t stack_flags, stack_cap, stack_end;
  size_t sync, sync_words, slots, logits, sg_logit, idx, w, sg, xperm, chunk_counts, chunk_masks, rank, counts, offsets, perm, inv,
      ptok, tiles, n_tiles, ticket, act, act_s, o, h, wnorm, xsum, asum, asum_s, total;
};

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Tiles of at most mt rows over the experts a step selects: sum_e
// ceil(c_e / mt) <= (T*k + (mt - 1) * min(T*k, E)) / mt, plus the shared
// expert's ceil(T / mt).
int max_tiles_bound(const ainfer_moe_shape &s, int T, int mt) {
  long tk = (long)T * s.top_k;
  long used = tk < s.n_experts ? tk : s.n_experts;
  long routed = (tk + (mt - 1) * used + mt - 1) / mt;
  long sh = s.shared_inter > 0 ? (T + mt - 1) / mt : 0;
  return (int)(routed + sh);
}

Layout layout_of(const ainfer_moe_shape &s, int Tm) {
  Layout L;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    size_t o = off;
    off += align256(bytes);
    return o;
  };
  const size_t T = (size_t)(Tm > 0 ? Tm : 1), E = s.n_experts, k = s.top_k, H = s.hidden;
  const size_t nchunks = (T + 63) / 64;
  // decode sync region: the same place and size for every T
  {
    DecodeGeom g;
    const int slabs = decode_geometry(s, &g) ? g.slabs_dn : 0;
    L.slots = SY_TILES + SY_STRIDE * (2 * (size_t)max_tiles_bound(s, DECODE_MAX_T, DEC_MT) +
                                      (size_t)DECODE_MAX_T * slabs);  // in words
    L.sync_words = L.slots + (size_t)DECODE_MAX_T * (E + 1);
    L.sync = take(L.sync_words * 4);
  }
  // the decode-stack kernel's tagged logit slots and item flags: also the
  // same place for every T, zeroed with the sync region
  L.stack_cap = (size_t)max_tiles_bound(s, DECODE_NORM_MAX_T, DEC_MT);
  L.stack_flags = take((size_t)stack_flag_words(s, (int)L.stack_cap) * 4);
  L.stack_end = off;
  L.logits = take(T * E * 4);
  L.sg_logit = take(T * 4);
  L.idx = take(T * k * 4);
  L.w = take(T * k * 4);
  L.sg = take(T * 4);
  L.xperm = take(T * H * 2);
  L.chunk_counts = take(nchunks * E * 4);
  L.chunk_masks = take(nchunks * E * 8);  // right after the counts: zeroed as one range
  L.rank = take(T * k * 4);
  L.counts = take(E * 4);
  L.offsets = take((E + 1) * 4);
  L.perm = take(T * k * 4);
  L.inv = take(T * k * 4);
  L.ptok = take(T * k * 4);
  L.tiles = take((size_t)max_tiles_bound(s, (int)T, DEC_MT) * 16);  // >= every other bound
  L.n_tiles = take(4);
  L.ticket = take(4);
  L.act = take(T * k * s.inter * 2);
  L.act_s = take(T * (size_t)(s.shared_inter > 0 ? s.shared_inter : 1) * 2);
  L.o = take(T * (k + 1) * H * 2);
  L.h = take(T * H * 2);
  L.wnorm = take(E * 4);
  L.xsum = take(T * (H / 128) * 4);
  L.asum = take(T * k * (s.inter / 128) * 4);
  L.asum_s = take(T * (size_t)(s.shared_inter > 0 ? s.shared_inter / 128 : 1) * 4);
  L.w8_xq = L.w8_xs = L.w8_act = L.w8_acts = L.w8_aq = L.w8_as = L.w8_aqs = L.w8_ass = L.w8_o = 0;
  if (s.precision == AINFER_PRECISION_W4A8) {
    const size_t Is = s.shared_inter > 0 ? s.shared_inter : 128, I = s.inter;
    L.w8_xq = take(T * H);
    L.w8_xs = take(T * (H / 128) * 4);
    L.w8_act = take(T * k * I * 4);
    L.w8_acts = take(T * Is * 4);
    L.w8_aq = take(T * k * I);
    L.w8_as = take(T * k * (I / 128) * 4);
    L.w8_aqs = take(T * Is);
    L.w8_ass = take(T * (Is / 128) * 4);
    L.w8_o = take(T * (k + 1) * H * 4);
  }
  L.total = off;
  return L;
}

template <typename P>
P *at(void *ws, size_t off) {
  return (P *)((char *)ws + off);
}

// Calls above AINFER_MOE_CHUNK_TOKENS tokens run as consecutive chunks of at
// most that many tokens on one workspace (the chunked prefill of the
// reference's recorded ChunkGemm lists): the workspace and every buffer offset
// stay those of one chunk.  Each token's routing and expert rows are computed
// within its chunk.
constexpr int CHUNK = AINFER_MOE_CHUNK_TOKENS;
int chunk_of(int T) { return T < CHUNK ? T : CHUNK; }

int check_ws(const ainfer_moe_shape *s, int T, void *ws, size_t ws_bytes) {
  if (!ws) return AINFER_ERR_NULL;
  if (((uintptr_t)ws) & 255) return AINFER_ERR_WORKSPACE;
  if (ws_bytes < layout_of(*s, T).total) return AINFER_ERR_WORKSPACE;
  return AINFER_OK;
}

int check_weights(const ainfer_moe_shape *s, const ainfer_moe_weights *w) {
  if (!w || !w->router_w || !w->w_gate || !w->s_gate || !w->w_up || !w->s_up || !w->w_down ||
      !w->s_down)
    return AINFER_ERR_NULL;
  if (s->shared_inter > 0 && (!w->ws_gate || !w->ss_gate || !w->ws_up || !w->ss_up ||
                              !w->ws_down || !w->ss_down))
    return AINFER_ERR_NULL;
  // 16-byte vector loads of weights, 8-byte loads of scale runs
  auto mis = [](const void *p, uintptr_t a) { return p && ((uintptr_t)p & (a - 1)); };
  if (mis(w->w_gate, 16) || mis(w->w_up, 16) || mis(w->w_down, 16) || mis(w->ws_gate, 16) ||
      mis(w->ws_up, 16) || mis(w->ws_down, 16) || mis(w->router_w, 16) ||
      mis(w->shared_gate_w, 16) || mis(w->s_gate, 8) || mis(w->s_up, 8) || mis(w->s_down, 8) ||
      mis(w->ss_gate, 8) || mis(w->ss_up, 8) || mis(w->ss_down, 8))
    return AINFER_ERR_ARG;
  return AINFER_OK;
}

#define HIP_TRY(expr)                              \
  do {                                             \
    if ((expr) != hipSuccess) return AINFER_ERR_HIP; \
  } while (0)
#define HIP_TRY_RC(expr)          \
  do {                            \
    const int rc_ = (expr);       \
    if (rc_ != AINFER_OK) return rc_; \
  } while (0)

DispatchOut dispatch_out(const ainfer_moe_shape *s, const Layout &L, void *ws, int T) {
  DispatchOut d;
  d.counts = at<int32_t>(ws, L.counts);
  d.offsets = at<int32_t>(ws, L.offsets);
  d.perm = at<int32_t>(ws, L.perm);
  d.inv = at<int32_t>(ws, L.inv);
  d.ptok = at<int32_t>(ws, L.ptok);
  d.tiles = at<int4>(ws, L.tiles);
  d.n_tiles = at<int32_t>(ws, L.n_tiles);
  d.ticket = at<int32_t>(ws, L.ticket);
  d.mt = DEC_MT;
  return d;
}

// Arguments of the small-tile expert kernels: mode 0 = gate/up (+ SiLU), mode
// 1 = down.
ExpertArgs expert_args(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const Layout &L,
                       void *ws, const DispatchOut &d, int T, int mode) {
  ExpertArgs a;
  memset(&a, 0, sizeof a);
  a.ptok = d.ptok;
  a.tiles = d.tiles;
  a.n_tiles = d.n_tiles;
  a.T = T;
  a.k = s->top_k;
  a.E = s->n_experts;
  a.H = s->hidden;
  a.I = s->inter;
  a.Is = s->shared_inter;
  if (mode == 0) {
    a.w0 = w->w_gate;
    a.w1 = w->w_up;
    a.s0 = (const uint16_t *)w->s_gate;
    a.s1 = (const uint16_t *)w->s_up;
    a.ws0 = w->ws_gate;
    a.ws1 = w->ws_up;
    a.ss0 = (const uint16_t *)w->ss_gate;
    a.ss1 = (const uint16_t *)w->ss_up;
    a.a_routed = at<uint16_t>(ws, L.xperm);
    a.a_shared = at<uint16_t>(ws, L.xperm);
    a.act = at<uint16_t>(ws, L.act);
    a.act_s = at<uint16_t>(ws, L.act_s);
  } else {
    a.w0 = w->w_down;
    a.s0 = (const uint16_t *)w->s_down;
    a.ws0 = w->ws_down;
    a.ss0 = (const uint16_t *)w->ss_down;
    a.a_routed = at<uint16_t>(ws, L.act);
    a.a_shared = at<uint16_t>(ws, L.act_s);
    a.o = at<uint16_t>(ws, L.o);
  }
  return a;
}

// norm (decode path only, ainfer_moe_block_forward): x is the residual stream and
// the routing kernel applies the RMSNorm itself
int down_kbw(const ainfer_moe_shape &s) { return down_kbw_of(s); }

// The layer in W4A8 (AINFER_PRECISION_W4A8): routing as in W4A16, with x
// quantized beside it, then the expert GEMVs of the reference's numerics.
//  T <= 16  the decode routing kernel (with norm the block's RMSNorm), tiles of
//           DEC_MT tokens
//  above    the staged router (k_select quantizes x), tiles of gemm_mt tokens
// Gate/up: the one-token GEMVs at T = 1 (moe_w4a8.hip), the int8 GEMM where
// w4a8_gemm_at (moe_gemm_w4a8.hip; it quantizes act), else the 16-row GEMV
// blocks.  Down: with the combine in one launch up to DC_MAX_T tokens (sizes to
// W8DC_MAX_K), else as gate/up with the fp32 combine.
int do_forward_w4a8(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *x,
                    const void *resid, void *y, int T, void *ws, hipStream_t st, ProfCall *pc,
                    const NormIn *norm = nullptr) {
  const Layout L = layout_of(*s, T);
  const int E = s->n_experts, k = s->top_k, H = s->hidden, I = s->inter, Is = s->shared_inter;
  const int has_shared = Is > 0;
  const bool decode = T <= DECODE_MAX_T, gemm = w4a8_gemm_at(*s, T);
  if (norm && !decode) return AINFER_ERR_ARG;  // the caller normalizes above that
  DispatchOut d = dispatch_out(s, L, ws, T);
  d.mt = decode ? DEC_MT : gemm_mt(*s, T);
  // the group sums take the places of the W4A16 GEMM's (the same counts of
  // 4-byte values)
  W8Rows xq, aq, aqs;
  xq.q = at<int8_t>(ws, L.w8_xq);
  xq.s = at<float>(ws, L.w8_xs);
  xq.sum = gemm ? at<int32_t>(ws, L.xsum) : nullptr;
  aq.q = at<int8_t>(ws, L.w8_aq);
  aq.s = at<float>(ws, L.w8_as);
  aq.sum = at<int32_t>(ws, L.asum);
  aqs.q = at<int8_t>(ws, L.w8_aqs);
  aqs.s = at<float>(ws, L.w8_ass);
  aqs.sum = at<int32_t>(ws, L.asum_s);
  int32_t *sync = at<int32_t>(ws, L.sync);
  if (decode) {
    DispatchOut dr = d;  // nothing here reads the per-expert counts or offsets
    dr.counts = nullptr;
    dr.offsets = nullptr;
    HIP_TRY(launch_route_decode(x, w->router_w, w->router_bias, w->shared_gate_w,
                                at<float>(ws, L.logits), at<float>(ws, L.sg_logit),
                                at<int32_t>(ws, L.idx), at<float>(ws, L.w), at<float>(ws, L.sg),
                                nullptr, T, H, E, k, has_shared, &dr, sync,
                                (uint32_t *)(sync + L.slots), norm, st, xq));
  } else {
    const bool fused = T <= FUSED_DISPATCH_MAX_T;
    unsigned long long *cmask =
        T >= GEMM_MIN_T ? at<unsigned long long>(ws, L.chunk_masks) : nullptr;
    HIP_TRY(launch_router_fast(x, w->router_w, w->router_bias, w->shared_gate_w,
                               at<float>(ws, L.logits), at<float>(ws, L.wnorm),
                               at<int32_t>(ws, L.idx), at<float>(ws, L.w), at<float>(ws, L.sg),
                               nullptr, nullptr, T, H, E, k, has_shared, fused ? &d : nullptr, st,
                               cmask ? at<int32_t>(ws, L.chunk_counts) : nullptr, cmask, xq));
    pc->end(2);
    if (!fused)
      HIP_TRY(launch_dispatch(at<int32_t>(ws, L.idx), T, k, E, d.mt, has_shared,
                              at<int32_t>(ws, L.chunk_counts), at<int32_t>(ws, L.rank), d, st,
                              cmask));
  }
  pc->end(3);
  const int mtb = max_tiles_bound(*s, T, d.mt);
  float *o = at<float>(ws, L.w8_o);
  W8GemmArgs g;  // the GEMM's, and the one-token kernels'
  memset(&g, 0, sizeof g);
  W4A8Args a;
  memset(&a, 0, sizeof a);
  g.x = xq;
  g.act = aq;
  g.act_s = aqs;
  a.xq = xq.q;
  a.xs = xq.s;
  a.act = at<float>(ws, L.w8_act);
  a.act_s = at<float>(ws, L.w8_acts);
  a.aq = aq.q;
  a.as = aq.s;
  a.aq_s = aqs.q;
  a.as_s = aqs.s;
  auto set = [&](auto &q, const void *w0, const void *s0, const void *w1, const void *s1,
                 const void *ws0, const void *ss0, const void *ws1, const void *ss1) {
    q.o = o;
    q.ptok = d.ptok;
    q.tiles = d.tiles;
    q.n_tiles = d.n_tiles;
    q.T = T;
    q.k = k;
    q.E = E;
    q.H = H;
    q.I = I;
    q.Is = Is;
    q.w0 = (const uint8_t *)w0;
    q.s0 = (const uint16_t *)s0;
    q.w1 = (const uint8_t *)w1;
    q.s1 = (const uint16_t *)s1;
    q.ws0 = (const uint8_t *)ws0;
    q.ss0 = (const uint16_t *)ss0;
    q.ws1 = (const uint8_t *)ws1;
    q.ss1 = (const uint16_t *)ss1;
  };
  auto gate_up = [&](auto &q) {
    set(q, w->w_gate, w->s_gate, w->w_up, w->s_up, w->ws_gate, w->ss_gate, w->ws_up, w->ss_up);
  };
  auto down = [&](auto &q) {
    set(q, w->w_down, w->s_down, nullptr, nullptr, w->ws_down, w->ss_down, nullptr, nullptr);
  };
  if (gemm) {
    gate_up(g);
    HIP_TRY(launch_w4a8_gemm(0, s->scale_dtype, g, mtb, st));
  } else {
    gate_up(a);
    HIP_TRY(T == 1 ? launch_w4a8_expert_t1(0, s->scale_dtype, a, mtb, st)
                   : launch_w4a8_expert(0, s->scale_dtype, a, mtb, st));
  }
  pc->end(4);
  down(a);
  if (T <= DC_MAX_T && (T == 1 || gemm) && I <= W8DC_MAX_K && Is <= W8DC_MAX_K) {
    HIP_TRY(launch_w4a8_down_combine(s->scale_dtype, a, aq, aqs, at<float>(ws, L.w),
                                     at<float>(ws, L.sg), d.inv, resid, y, sync + SY_ERR, st));
    pc->end(5);
    return AINFER_OK;
  }
  if (gemm) {
    down(g);
    HIP_TRY(launch_w4a8_gemm(1, s->scale_dtype, g, mtb, st));
  } else {
    HIP_TRY(T == 1 ? launch_w4a8_expert_t1(1, s->scale_dtype, a, mtb, st)
                   : launch_w4a8_expert(1, s->scale_dtype, a, mtb, st));
  }
  pc->end(5);
  HIP_TRY(launch_combine_f32(o, d.inv, at<float>(ws, L.w), at<float>(ws, L.sg), has_shared, resid,
                             y, T, k, H, sync + SY_ERR, st));
  pc->end(6);
  return AINFER_OK;
}

// The expert stage on the dispatch d in the workspace, x in MFMA order
// written (and its group sums where gemm): the grouped GEMM, else the
// streaming items over tiles of DEC_MT tokens.  Leaves o in the workspace: dispatch-position rows,
// the shared expert's at rows T * k + t.
int run_experts(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const Layout &L,
                void *ws, DispatchOut &d, int T, bool gemm, hipStream_t st, ProfCall *pc) {
  const int E = s->n_experts, k = s->top_k, H = s->hidden;
  if (gemm) {
    GemmArgs g;
    memset(&g, 0, sizeof g);
    g.ptok = d.ptok;
    g.tiles = d.tiles;
    g.n_tiles = d.n_tiles;
    g.T = T;
    g.k = k;
    g.E = E;
    g.H = H;
    g.I = s->inter;
    g.Is = s->shared_inter;
    g.xsum = at<float>(ws, L.xsum);
    g.asum = at<float>(ws, L.asum);
    g.asum_s = at<float>(ws, L.asum_s);
    const int gtiles = max_tiles_bound(*s, T, d.mt);
    g.w0 = w->w_gate;
    g.w1 = w->w_up;
    g.s0 = (const uint16_t *)w->s_gate;
    g.s1 = (const uint16_t *)w->s_up;
    g.ws0 = w->ws_gate;
    g.ws1 = w->ws_up;
    g.ss0 = (const uint16_t *)w->ss_gate;
    g.ss1 = (const uint16_t *)w->ss_up;
    g.a_routed = at<uint16_t>(ws, L.xperm);
    g.act = at<uint16_t>(ws, L.act);
    g.act_s = at<uint16_t>(ws, L.act_s);
    HIP_TRY(launch_expert_gemm(0, s->scale_dtype, g, gtiles, st));
    pc->end(4);
    g.w0 = w->w_down;
    g.s0 = (const uint16_t *)w->s_down;
    g.ws0 = w->ws_down;
    g.ss0 = (const uint16_t *)w->ss_down;
    g.w1 = nullptr;
    g.s1 = nullptr;
    g.ws1 = nullptr;
    g.ss1 = nullptr;
    g.a_routed = at<uint16_t>(ws, L.act);
    g.a_shared = at<uint16_t>(ws, L.act_s);
    g.o = at<uint16_t>(ws, L.o);
    HIP_TRY(launch_expert_gemm(1, s->scale_dtype, g, gtiles, st));
    pc->end(5);
    return AINFER_OK;
  }
  ExpertArgs a;
  memset(&a, 0, sizeof a);
  a.ptok = d.ptok;
  a.tiles = d.tiles;
  a.n_tiles = d.n_tiles;
  a.T = T;
  a.k = k;
  a.E = E;
  a.H = H;
  a.I = s->inter;
  a.Is = s->shared_inter;
  const int smt = DEC_MT;  // tiles of the dispatch above
  const int max_tiles = max_tiles_bound(*s, T, smt);
  // k-groups per wave and 16-row groups per wave, measured at T = 1, 4, 16
  const int kbw = 4, kbw_down = down_kbw(*s);
  // gate/up + SiLU-mul
  a.w0 = w->w_gate;
  a.w1 = w->w_up;
  a.s0 = (const uint16_t *)w->s_gate;
  a.s1 = (const uint16_t *)w->s_up;
  a.ws0 = w->ws_gate;
  a.ws1 = w->ws_up;
  a.ss0 = (const uint16_t *)w->ss_gate;
  a.ss1 = (const uint16_t *)w->ss_up;
  a.a_routed = at<uint16_t>(ws, L.xperm);
  a.a_shared = at<uint16_t>(ws, L.xperm);
  a.act = at<uint16_t>(ws, L.act);
  a.act_s = at<uint16_t>(ws, L.act_s);
  HIP_TRY(launch_expert_stream(0, s->scale_dtype, a, max_tiles, kbw, st));
  pc->end(4);
  // down + combine
  a.w0 = w->w_down;
  a.s0 = (const uint16_t *)w->s_down;
  a.ws0 = w->ws_down;
  a.ss0 = (const uint16_t *)w->ss_down;
  a.w1 = nullptr;
  a.s1 = nullptr;
  a.ws1 = nullptr;
  a.ss1 = nullptr;
  a.a_routed = at<uint16_t>(ws, L.act);
  a.a_shared = at<uint16_t>(ws, L.act_s);
  a.o = at<uint16_t>(ws, L.o);
  HIP_TRY(launch_expert_stream(1, s->scale_dtype, a, max_tiles, kbw_down, st));
  pc->end(5);
  return AINFER_OK;
}

int do_forward(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *x,
               const void *resid, void *y, int T, void *ws, hipStream_t st,
               ProfCall *pc, const NormIn *norm = nullptr, const NormIn *next = nullptr,
               void *h_next = nullptr) {
  // the final combine, or (next non-null, W4A16, resid non-null) the combine
  // followed by the next block's RMSNorm of the rows it writes, into h_next
  auto combine = [&](const DispatchOut &d, const Layout &L) -> hipError_t {
    if (next && resid)
      return launch_combine_norm(at<uint16_t>(ws, L.o), d.inv, at<float>(ws, L.w),
                                 at<float>(ws, L.sg), s->shared_inter > 0, resid, y, T,
                                 s->top_k, s->hidden, at<int32_t>(ws, L.sync) + SY_ERR, *next,
                                 h_next, st);
    return launch_combine(at<uint16_t>(ws, L.o), d.inv, at<float>(ws, L.w), at<float>(ws, L.sg),
                          s->shared_inter > 0, resid, y, T, s->top_k, s->hidden,
                          at<int32_t>(ws, L.sync) + SY_ERR, st);
  };
  if (s->precision == AINFER_PRECISION_W4A8)
    return do_forward_w4a8(s, w, x, resid, y, T, ws, st, pc, norm);
  const Layout L = layout_of(*s, T);
  const int E = s->n_experts, k = s->top_k, H = s->hidden;
  const int has_shared = s->shared_inter > 0;
  const bool fused = T <= FUSED_DISPATCH_MAX_T;
  const bool gemm = expert_gemm_at(*s, T);
  const int mt = gemm ? gemm_mt(*s, T) : DEC_MT;
  DispatchOut d = dispatch_out(s, L, ws, T);
  d.mt = mt;
  DecodeGeom dg;
  if (T <= DECODE_MAX_T) {
    // decode: the routing kernel, then two or three expert launches
    int32_t *sync = at<int32_t>(ws, L.sync);
    // the expert kernels read the tiles and positions only: no per-expert
    // counts or offsets on this path
    DispatchOut dr = d;
    dr.counts = nullptr;
    dr.offsets = nullptr;
    HIP_TRY(launch_route_decode(x, w->router_w, w->router_bias, w->shared_gate_w,
                                at<float>(ws, L.logits), at<float>(ws, L.sg_logit),
                                at<int32_t>(ws, L.idx), at<float>(ws, L.w), at<float>(ws, L.sg),
                                at<uint16_t>(ws, L.xperm), T, H, E, k, has_shared, &dr, sync,
                                (uint32_t *)(sync + L.slots), norm, st));
    pc->end(2);
    ExpertArgs gu = expert_args(s, w, L, ws, d, T, 0), dn = expert_args(s, w, L, ws, d, T, 1);
    const int mtb = max_tiles_bound(*s, T, DEC_MT);
    const int kbw_dn = T <= FUSED_EXPERTS_MAX_T ? 2 : down_kbw(*s);
    if (T == FUSED_EXPERTS_MAX_T && !down_combine_at(*s, T) && decode_geometry(*s, &dg)) {
      // latency-bound: gate/up, down and combine in one launch
      HIP_TRY(launch_experts_decode(s->scale_dtype, dg, gu, dn, at<float>(ws, L.w),
                                    at<float>(ws, L.sg), d.inv, resid, y, sync, mtb,
                                    max_tiles_bound(*s, DECODE_MAX_T, DEC_MT), st));
      pc->end(5);
      return AINFER_OK;
    }
    pc->kernel_events();
    HIP_TRY(launch_expert_stream(0, s->scale_dtype, gu, mtb, 4, st));
    pc->end(4);
    if (down_combine_at(*s, T)) {
      int kbw, wk, wr;
      if (!expert_geometry(1, H, s->inter, s->shared_inter, kbw_dn, &kbw, &wk, &wr))
        return AINFER_ERR_SHAPE;
      HIP_TRY(launch_down_combine(s->scale_dtype, dn, kbw, at<float>(ws, L.w),
                                  at<float>(ws, L.sg), d.inv, resid, y, sync + SY_ERR, st));
      pc->end(5);
      return AINFER_OK;
    }
    HIP_TRY(launch_expert_stream(1, s->scale_dtype, dn, mtb, kbw_dn, st));
    pc->end(5);
    HIP_TRY(combine(d, L));
    pc->end(6);
    return AINFER_OK;
  }
  // prefill (T >= GEMM_MIN_T, unfused dispatch): the selection builds the
  // dispatch's per-chunk token masks itself, so the dispatch needs no counting launch
  unsigned long long *cmask =
      T >= GEMM_MIN_T ? at<unsigned long long>(ws, L.chunk_masks) : nullptr;
  HIP_TRY(launch_router_fast(x, w->router_w, w->router_bias, w->shared_gate_w,
                               at<float>(ws, L.logits), at<float>(ws, L.wnorm),
                               at<int32_t>(ws, L.idx), at<float>(ws, L.w), at<float>(ws, L.sg),
                               at<uint16_t>(ws, L.xperm), gemm ? at<float>(ws, L.xsum) : nullptr,
                               T, H, E, k, has_shared, fused ? &d : nullptr, st,
                               cmask ? at<int32_t>(ws, L.chunk_counts) : nullptr, cmask));
  pc->end(2);
  if (!fused)
    HIP_TRY(launch_dispatch(at<int32_t>(ws, L.idx), T, k, E, mt, has_shared,
                            at<int32_t>(ws, L.chunk_counts), at<int32_t>(ws, L.rank), d, st,
                            cmask));
  pc->end(3);
  HIP_TRY_RC(run_experts(s, w, L, ws, d, T, gemm, st, pc));
  HIP_TRY(combine(d, L));
  pc->end(6);
  return AINFER_OK;
}

int check_block_args(const ainfer_moe_shape *s, const ainfer_moe_weights *w, int norm_mode,
                     float eps, const void *resid_in, const void *resid_out, int T) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if ((rc = check_weights(s, w))) return rc;
  if (norm_mode != AINFER_NORM_PLAIN && norm_mode != AINFER_NORM_ONE_PLUS) return AINFER_ERR_ARG;
  if (!(eps >= 0.0f)) return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if (!resid_in || !resid_out) return AINFER_ERR_NULL;
  return AINFER_OK;
}

// h = RMSNorm(resid_in); resid_out = resid_in + MoE(h), on a checked workspace
int do_block(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *norm_w,
             int norm_mode, float eps, const void *resid_in, void *resid_out, int T, void *ws,
             hipStream_t st) {
  const Layout L = layout_of(*s, T);
  void *h = at<void>(ws, L.h);
  ProfCall pc(st);
  pc.start();
  if (T <= DECODE_NORM_MAX_T) {
    // decode at up to 4 tokens: the routing kernel normalizes x itself (one
    // launch fewer per block: c4 T=1 about 2470 -> 2235 us per 60-block
    // step); the values are those k_rmsnorm writes
    NormIn n;
    n.w = (const uint16_t *)norm_w;
    n.mode = norm_mode;
    n.eps = eps;
    n.on = 1;
    pc.end(0);
    return do_forward(s, w, resid_in, resid_in, resid_out, T, ws, st, &pc, &n);
  }
  HIP_TRY(launch_rmsnorm(resid_in, norm_w, norm_mode, eps, h, T, s->hidden, st));
  pc.end(0);
  return do_forward(s, w, h, resid_in, resid_out, T, ws, st, &pc);
}

// ---- the no-allocation entry's scratch ---------------------------------------
// One copy per GPU, alive until the process ends.  Host code must never pass
// the array's name to a kernel or a copy (on the host it is only a stand-in
// symbol); it uses the per-device address hipGetSymbolAddress returns.
__device__ __align__(256) unsigned char scratch[AINFER_MOE_NOALLOC_SCRATCH_BYTES];

// host copies of the tables ainfer_moe_stack_prepare wrote, by device address
std::mutex g_tables_mu;
std::map<const void *, std::vector<StackLayer>> g_tables;

constexpr int NOALLOC_MAX_DEVICES = 64;
std::mutex g_scratch_mu;
void *g_scratch_ptr[NOALLOC_MAX_DEVICES];

// The current device's scratch address, looked up once per device.
int noalloc_scratch(void **out) {
  int dev = -1;
  HIP_TRY(hipGetDevice(&dev));
  if (dev < 0 || dev >= NOALLOC_MAX_DEVICES) return AINFER_ERR_HIP;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void *p = nullptr;
    HIP_TRY(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
    if (!p || ((uintptr_t)p & 255)) return AINFER_ERR_HIP;
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return AINFER_OK;
}

}  // namespace

namespace {
int do_route(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *x, int T,
             int32_t *topk_idx, float *topk_w, float *shared_gate, float *logits, void *ws,
             hipStream_t st) {
  const Layout L = layout_of(*s, T);
  if (T <= DECODE_MAX_T) {
    // the decode routing kernel, without its dispatch
    HIP_TRY(launch_route_decode(x, w->router_w, w->router_bias, w->shared_gate_w,
                                logits ? logits : at<float>(ws, L.logits),
                                at<float>(ws, L.sg_logit), topk_idx, topk_w, shared_gate, nullptr,
                                T, s->hidden, s->n_experts, s->top_k, s->shared_inter > 0,
                                nullptr, at<int32_t>(ws, L.sync),
                                at<uint32_t>(ws, L.sync) + L.slots, nullptr, st));
    return AINFER_OK;
  }
  HIP_TRY(launch_router_fast(x, w->router_w, w->router_bias, w->shared_gate_w,
                             at<float>(ws, L.logits), at<float>(ws, L.wnorm), topk_idx, topk_w,
                             shared_gate, nullptr, nullptr, T, s->hidden, s->n_experts,
                             s->top_k, s->shared_inter > 0, nullptr, st));
  // the full canonical logits, on request (lane-strided chunk order, VALU)
  if (logits)
    HIP_TRY(launch_router(x, w->router_w, w->router_bias, w->shared_gate_w, logits,
                          at<float>(ws, L.sg_logit), nullptr, T, s->hidden, s->n_experts, st));
  return AINFER_OK;
}

// ---- the operators around the expert stage ----------------------------------
bool mis(const void *p, uintptr_t align) { return ((uintptr_t)p & (align - 1)) != 0; }
bool is_act(int32_t dtype) { return dtype == AINFER_ACT_F32 || dtype == AINFER_ACT_BF16; }
int act_size(int32_t dtype) { return dtype == AINFER_ACT_F32 ? 4 : 2; }
// two runs of bytes with one in common
bool meet(const void *p, size_t n, const void *q, size_t m) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && (a < b ? b - a < n : a - b < m);
}
// row pitches (in elements) whose products with a token count stay far from 2^63
constexpr int64_t MAX_LD = (int64_t)1 << 40;

int check_lora(const ainfer_moe_lora *l) {
  if (!l) return AINFER_ERR_NULL;
  if (l->n_adapters < 1 || l->n_adapters > 4096 || l->rank < 8 || l->rank > 128 || l->rank % 8 ||
      l->in < 8 || l->in > 65536 || l->in % 8 || l->n_proj < 1 ||
      l->n_proj > AINFER_LORA_MAX_PROJ)
    return AINFER_ERR_SHAPE;
  for (int p = 0; p < l->n_proj; ++p)
    if (l->out[p] < 1 || l->out[p] > (1 << 20)) return AINFER_ERR_SHAPE;
  if (!is_act(l->x_dtype) || !is_act(l->y_dtype)) return AINFER_ERR_ARG;
  return AINFER_OK;
}

// ---- experts in 8-bit floating point, tokens sorted by expert ------------------
// the same for up to AINFER_MOE_MAX_ROWS rows
constexpr int64_t MAX_ROW_LD = (int64_t)1 << 36;
bool is_scale_kind(int32_t kind) {
  return kind == AINFER_FP8_SCALE_ANY || kind == AINFER_FP8_SCALE_POW2;
}
// a pitch that fits rows of `cols` elements
bool bad_ld(int64_t ld, int64_t cols) { return ld < cols || ld > MAX_ROW_LD; }
// `rows` rows of `cols` elements as bytes; rows without room between them are one row
struct ByteRows {
  intptr_t at;
  int64_t n, pitch, bytes;
};
ByteRows byte_rows(const void *p, int64_t rows, int64_t ld, int64_t cols, int size) {
  if (rows == 1 || ld == cols) return {(intptr_t)p, rows > 0, rows * cols * size, rows * cols * size};
  return {(intptr_t)p, rows, ld * size, cols * size};
}
// whether a row of r meets [at, at + n): the first row that ends behind `at` starts ahead of its end
bool rows_meet(const ByteRows &r, intptr_t at, int64_t n) {
  const intptr_t end = r.at + r.bytes;
  if (r.n < 2 || n == 0) return r.n && n && at < end && r.at < at + n;
  const int64_t i = at < end ? 0 : (at - end) / r.pitch + 1;
  return i < r.n && r.at + i * r.pitch < at + n;
}
// Whether rows that are written meet n bytes at p.
bool over(const void *out, int64_t rows, int64_t ld, int64_t cols, int size, const void *p,
          size_t n) {
  return out && p && rows_meet(byte_rows(out, rows, ld, cols, size), (intptr_t)p, (int64_t)n);
}
// Whether rows that are written meet other rows.  With rows of both pitched, and differently, each
// one's first row is looked for among the other's.
bool over_rows(const void *out, int64_t rows, int64_t ld, int64_t cols, int size, const void *in,
               int64_t in_rows, int64_t in_ld, int64_t in_cols, int in_size) {
  if (!out || !in) return false;
  const ByteRows a = byte_rows(out, rows, ld, cols, size),
                 b = byte_rows(in, in_rows, in_ld, in_cols, in_size);
  if (a.n > 1 && b.n > 1 && a.pitch == b.pitch) {
    // row j of b is d + (j - i) pitch from row i of a: the least such distance above -b.bytes
    const int64_t d = b.at - a.at, low = -b.bytes - d;
    const int64_t below = low / a.pitch - (low % a.pitch < 0);
    const int64_t m = std::max(below + 1, 1 - a.n);
    return m < b.n && d + m * a.pitch < a.bytes;
  }
  return (b.n && rows_meet(a, b.at, b.bytes)) || (a.n && rows_meet(b, a.at, a.bytes));
}
int check_fp8_sizes(int32_t E, int32_t M, int32_t K) {
  if (E < 1 || E > 1024 || M < 1 || M > (1 << 20) || K < 16 || K > 65536 || K % 16 ||
      (int64_t)E * M * K > (int64_t)1 << 38)
    return AINFER_ERR_SHAPE;
  return AINFER_OK;
}
int check_fp8(const ainfer_moe_fp8 *w) {
  if (!w) return AINFER_ERR_NULL;
  int rc = check_fp8_sizes(w->n_experts, w->rows, w->cols);
  if (rc) return rc;
  return is_act(w->y_dtype) ? AINFER_OK : AINFER_ERR_ARG;
}
int check_sorting(const ainfer_moe_sorting *s) {
  if (!s) return AINFER_ERR_NULL;
  if (s->n_experts < 1 || s->n_experts > 1024 || s->top_k < 1 || s->top_k > 32 ||
      s->hidden < 1 || s->hidden > 65536 || (s->fp8 && s->hidden % 16))
    return AINFER_ERR_SHAPE;
  if (!is_act(s->x_dtype) || (s->fp8 != 0 && s->fp8 != 1) || !is_scale_kind(s->scale_kind))
    return AINFER_ERR_ARG;
  return AINFER_OK;
}
}  // namespace

extern "C" {

const char *ainfer_moe_strerror(int status) {
  switch (status) {
  case AINFER_OK: return "ok";
  case AINFER_ERR_SHAPE: return "unsupported shape";
  case AINFER_ERR_NULL: return "required pointer is NULL";
  case AINFER_ERR_WORKSPACE: return "workspace too small or not 256-byte aligned";
  case AINFER_ERR_TOKENS: return "token count out of range";
  case AINFER_ERR_HIP: return "HIP runtime error";
  case AINFER_ERR_ARG: return "argument out of range";
  case AINFER_ERR_SYNC: return "a device-side wait ran out (workspace synchronisation words)";
  case AINFER_ERR_SCRATCH:
    return "the call needs more workspace than the no-allocation entry's static scratch holds";
  default: return "unknown status";
  }
}

int ainfer_moe_validate(const ainfer_moe_shape *s) {
  if (!s) return AINFER_ERR_NULL;
  if (s->group != 128) return AINFER_ERR_SHAPE;
  if (s->precision != AINFER_PRECISION_W4A16 && s->precision != AINFER_PRECISION_W4A8)
    return AINFER_ERR_SHAPE;
  // K of every expert product <= 4096: the row kernels hold a row of 64 lanes x 8
  // chunks in registers, and the GEMMs' token offsets (T <= 4096 rows) are 32-bit
  if (s->hidden < 128 || s->hidden % 128 || s->hidden > 4096) return AINFER_ERR_SHAPE;
  if (s->inter < 128 || s->inter % 128 || s->inter > 4096) return AINFER_ERR_SHAPE;
  if (s->shared_inter < 0 || s->shared_inter % 128 || s->shared_inter > 4096)
    return AINFER_ERR_SHAPE;
  if (s->n_experts < 1 || s->n_experts > 1024) return AINFER_ERR_SHAPE;
  if (s->top_k < 1 || s->top_k > 32 || s->top_k > s->n_experts) return AINFER_ERR_SHAPE;
  if (s->scale_dtype != AINFER_SCALE_FP16 && s->scale_dtype != AINFER_SCALE_BF16)
    return AINFER_ERR_SHAPE;
  if (!router_supported(s->hidden, s->n_experts)) return AINFER_ERR_SHAPE;
  int kbw, wk, wr;
  for (int mode = 0; mode < 2; ++mode)
    if (!expert_geometry(mode, s->hidden, s->inter, s->shared_inter, 1, &kbw, &wk, &wr))
      return AINFER_ERR_SHAPE;
  return AINFER_OK;
}

size_t ainfer_moe_workspace_bytes(const ainfer_moe_shape *s, int32_t max_tokens) {
  if (ainfer_moe_validate(s) != AINFER_OK) return 0;
  if (max_tokens < 0 || max_tokens > AINFER_MOE_MAX_TOKENS) return 0;
  return layout_of(*s, chunk_of(max_tokens)).total;
}

int ainfer_moe_workspace_init(const ainfer_moe_shape *s, void *ws, size_t ws_bytes,
                              void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if ((rc = check_ws(s, 0, ws, ws_bytes))) return rc;
  const Layout L = layout_of(*s, 0);
  HIP_TRY(launch_zero_i32(at<int32_t>(ws, L.sync), (int)((L.stack_end - L.sync) / 4),
                          (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_workspace_check(const ainfer_moe_shape *s, const void *ws, size_t ws_bytes,
                               void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if ((rc = check_ws(s, 0, const_cast<void *>(ws), ws_bytes))) return rc;
  const Layout L = layout_of(*s, 0);
  std::vector<int32_t> h(L.sync_words);
  HIP_TRY(hipStreamSynchronize((hipStream_t)stream));
  HIP_TRY(hipMemcpy(h.data(), at<int32_t>(const_cast<void *>(ws), L.sync), L.sync_words * 4,
                    hipMemcpyDeviceToHost));
  if (h[SY_ERR]) return AINFER_ERR_SYNC;
  for (size_t i = 0; i < h.size(); ++i)
    if (h[i]) return AINFER_ERR_WORKSPACE;
  return AINFER_OK;
}

}  // extern "C"

namespace {
std::atomic<int> g_strict{0};

// Strict mode: wait for the call's work and report a bounded wait that ran
// out (the workspace's sticky error word).  rc: the call's own result so far.
int strict_finish(int rc, const void *ws, void *stream) {
  if (rc || !g_strict.load() || !ws) return rc;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  HIP_TRY(hipStreamIsCapturing((hipStream_t)stream, &cs));
  if (cs != hipStreamCaptureStatusNone) return AINFER_OK;
  HIP_TRY(hipStreamSynchronize((hipStream_t)stream));
  int32_t err = 0;
  // the sync region starts the workspace (layout_of: offset 0)
  HIP_TRY(hipMemcpy(&err, (const int32_t *)ws + SY_ERR, sizeof err, hipMemcpyDeviceToHost));
  return err ? AINFER_ERR_SYNC : AINFER_OK;
}
}  // namespace

extern "C" {

int ainfer_moe_set_strict(int32_t on) {
  g_strict.store(on ? 1 : 0);
  return AINFER_OK;
}

int ainfer_moe_forward(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *x,
                       void *y, int32_t T, void *ws, size_t ws_bytes, void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if ((rc = check_weights(s, w))) return rc;
  if (T == 0) return AINFER_OK;
  if (!x || !y) return AINFER_ERR_NULL;
  if ((rc = check_ws(s, chunk_of(T), ws, ws_bytes))) return rc;
  const size_t row = (size_t)s->hidden * 2;
  for (int t0 = 0; t0 < T; t0 += CHUNK) {
    ProfCall pc((hipStream_t)stream);
    pc.start();
    if ((rc = do_forward(s, w, (const char *)x + t0 * row, nullptr, (char *)y + t0 * row,
                         chunk_of(T - t0), ws, (hipStream_t)stream, &pc)))
      return rc;
  }
  return strict_finish(AINFER_OK, ws, stream);
}

int ainfer_moe_block_forward(const ainfer_moe_shape *s, const ainfer_moe_weights *w,
                             const void *norm_w, int32_t norm_mode, float eps,
                             const void *resid_in, void *resid_out, int32_t T, void *ws,
                             size_t ws_bytes, void *stream) {
  int rc = check_block_args(s, w, norm_mode, eps, resid_in, resid_out, T);
  if (rc || T == 0) return rc;
  if ((rc = check_ws(s, chunk_of(T), ws, ws_bytes))) return rc;
  const size_t row = (size_t)s->hidden * 2;
  for (int t0 = 0; t0 < T; t0 += CHUNK)
    if ((rc = do_block(s, w, norm_w, norm_mode, eps, (const char *)resid_in + t0 * row,
                       (char *)resid_out + t0 * row, chunk_of(T - t0), ws, (hipStream_t)stream)))
      return rc;
  return strict_finish(AINFER_OK, ws, stream);
}

int ainfer_moe_block_forward_noalloc(const ainfer_moe_shape *s, const ainfer_moe_weights *w,
                                     const void *norm_w, int32_t norm_mode, float eps,
                                     const void *resid_in, void *resid_out, int32_t T,
                                     void *stream) {
  int rc = check_block_args(s, w, norm_mode, eps, resid_in, resid_out, T);
  if (rc || T == 0) return rc;
  if (layout_of(*s, chunk_of(T)).total > AINFER_MOE_NOALLOC_SCRATCH_BYTES)
    return AINFER_ERR_SCRATCH;
  void *ws = nullptr;
  if ((rc = noalloc_scratch(&ws))) return rc;
  hipStream_t st = (hipStream_t)stream;
  // every call starts from zeroed synchronisation words (a fill kernel, so the
  // call stays capturable into a HIP graph): a bounded wait that ran out in
  // an earlier call (that call's outputs are NaN) leaves nothing behind
  const Layout L0 = layout_of(*s, 0);
  HIP_TRY(launch_zero_i32(at<int32_t>(ws, L0.sync), (int)L0.sync_words, st));
  const size_t row = (size_t)s->hidden * 2;
  for (int t0 = 0; t0 < T; t0 += CHUNK)
    if ((rc = do_block(s, w, norm_w, norm_mode, eps, (const char *)resid_in + t0 * row,
                       (char *)resid_out + t0 * row, chunk_of(T - t0), ws, st)))
      return rc;
  return strict_finish(AINFER_OK, ws, stream);
}

size_t ainfer_moe_stack_table_bytes(int32_t n_layers) {
  return n_layers > 0 ? (size_t)n_layers * sizeof(StackLayer) : 0;
}

int ainfer_moe_stack_prepare(const ainfer_moe_shape *s, const ainfer_moe_weights *layers,
                             const void *const *norm_w, int32_t n_layers, void *table,
                             size_t table_bytes, void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (n_layers <= 0) return AINFER_ERR_ARG;
  if (!layers || !table) return AINFER_ERR_NULL;
  if (((uintptr_t)table) & 15 || table_bytes < ainfer_moe_stack_table_bytes(n_layers))
    return AINFER_ERR_ARG;
  std::vector<StackLayer> h((size_t)n_layers);
  for (int l = 0; l < n_layers; ++l) {
    if ((rc = check_weights(s, &layers[l]))) return rc;
    memset(&h[l], 0, sizeof(StackLayer));
    h[l].w = layers[l];
    h[l].norm_w = norm_w ? norm_w[l] : nullptr;
    if (h[l].norm_w && ((uintptr_t)h[l].norm_w & 15)) return AINFER_ERR_ARG;
  }
  hipStream_t st = (hipStream_t)stream;
  HIP_TRY(hipMemcpyAsync(table, h.data(), h.size() * sizeof(StackLayer), hipMemcpyHostToDevice,
                         st));
  HIP_TRY(hipStreamSynchronize(st));
  // the host keeps its own copy for the replayed form, which launches the
  // layers' kernels from the host
  std::lock_guard<std::mutex> lock(g_tables_mu);
  g_tables[table] = std::move(h);
  return AINFER_OK;
}

size_t ainfer_moe_stack_workspace_bytes(const ainfer_moe_shape *s, int32_t max_tokens,
                                        int32_t n_layers) {
  if (ainfer_moe_validate(s) != AINFER_OK) return 0;
  if (max_tokens < 1 || max_tokens > AINFER_MOE_MAX_TOKENS || n_layers < 1) return 0;
  size_t need = layout_of(*s, chunk_of(max_tokens)).total;  // the replayed form
  StackGeom g;
  if (max_tokens <= DECODE_NORM_MAX_T && stack_geometry(*s, max_tokens, &g)) {
    const size_t p = layout_of(*s, 1).total + (size_t)n_layers * stack_layer_bytes(*s, max_tokens, nullptr);
    if (p > need) need = p;  // the persistent form's per-layer regions
  }
  return need;
}

namespace {
int check_stack_args(const ainfer_moe_shape *s, const void *table, int32_t n_layers,
                     int32_t norm_mode, float eps, const void *resid_in, const void *resid_out,
                     int32_t T, int max_t) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (T < 0 || T > max_t) return AINFER_ERR_TOKENS;
  if (n_layers < 0) return AINFER_ERR_ARG;
  if (norm_mode != AINFER_NORM_PLAIN && norm_mode != AINFER_NORM_ONE_PLUS) return AINFER_ERR_ARG;
  if (!(eps >= 0.0f)) return AINFER_ERR_ARG;
  if (T == 0 || n_layers == 0) return AINFER_OK;
  if (!table || !resid_in || !resid_out) return AINFER_ERR_NULL;
  if (((uintptr_t)table) & 15 || ((uintptr_t)resid_in) & 15 || ((uintptr_t)resid_out) & 15)
    return AINFER_ERR_ARG;
  return AINFER_OK;
}

// The replayed stack on one chunk of at most CHUNK tokens.  Where the block's
// routing kernel normalizes x itself (decode, T <= 4) and in W4A8, the layers
// are the per-block entry's calls as they are.  Elsewhere the first layer's
// RMSNorm is a launch of its own and every later one is computed by the
// previous layer's combine, from the rows it writes (launch_combine_norm),
// into the workspace's h; the values are those the block entry computes.
int do_stack(const ainfer_moe_shape *s, const std::vector<StackLayer> &ly, int n_layers,
             int norm_mode, float eps, const void *resid_in, void *resid_out, int T, void *ws,
             hipStream_t st) {
  const bool folded = T <= DECODE_NORM_MAX_T;
  if (folded || s->precision == AINFER_PRECISION_W4A8) {
    for (int l = 0; l < n_layers; ++l) {
      int rc = do_block(s, &ly[l].w, ly[l].norm_w, norm_mode, eps, l ? resid_out : resid_in,
                        resid_out, T, ws, st);
      if (rc) return rc;
    }
    return AINFER_OK;
  }
  const Layout L = layout_of(*s, T);
  void *h = at<void>(ws, L.h);
  for (int l = 0; l < n_layers; ++l) {
    ProfCall pc(st);
    pc.start();
    if (l == 0)
      HIP_TRY(launch_rmsnorm(resid_in, ly[0].norm_w, norm_mode, eps, h, T, s->hidden, st));
    pc.end(0);
    NormIn nx;
    nx.w = l + 1 < n_layers ? (const uint16_t *)ly[l + 1].norm_w : nullptr;
    nx.mode = norm_mode;
    nx.eps = eps;
    nx.on = 1;
    int rc = do_forward(s, &ly[l].w, h, l ? resid_out : resid_in, resid_out, T, ws, st, &pc,
                        nullptr, l + 1 < n_layers ? &nx : nullptr, h);
    if (rc) return rc;
  }
  return AINFER_OK;
}
}  // namespace

int ainfer_moe_stack_forward(const ainfer_moe_shape *s, const void *table, int32_t n_layers,
                             int32_t norm_mode, float eps, const void *resid_in,
                             void *resid_out, int32_t T, void *ws, size_t ws_bytes,
                             void *stream) {
  int rc = check_stack_args(s, table, n_layers, norm_mode, eps, resid_in, resid_out, T,
                            AINFER_MOE_MAX_TOKENS);
  if (rc || T == 0 || n_layers == 0) return rc;
  if ((rc = check_ws(s, chunk_of(T), ws, ws_bytes))) return rc;
  std::vector<StackLayer> ly;
  {
    std::lock_guard<std::mutex> lock(g_tables_mu);
    auto it = g_tables.find(table);
    if (it == g_tables.end() || (int)it->second.size() < n_layers) return AINFER_ERR_ARG;
    ly.assign(it->second.begin(), it->second.begin() + n_layers);
  }
  // tokens are independent through the whole stack: each chunk runs all layers
  const size_t row = (size_t)s->hidden * 2;
  for (int t0 = 0; t0 < T; t0 += CHUNK)
    if ((rc = do_stack(s, ly, n_layers, norm_mode, eps, (const char *)resid_in + t0 * row,
                       (char *)resid_out + t0 * row, chunk_of(T - t0), ws, (hipStream_t)stream)))
      return rc;
  return strict_finish(AINFER_OK, ws, stream);
}

int ainfer_moe_stack_forward_persistent(const ainfer_moe_shape *s, const void *table,
                                        int32_t n_layers, int32_t norm_mode, float eps,
                                        const void *resid_in, void *resid_out, int32_t T,
                                        void *ws, size_t ws_bytes, void *stream) {
  int rc = check_stack_args(s, table, n_layers, norm_mode, eps, resid_in, resid_out, T,
                            DECODE_NORM_MAX_T);
  if (rc || T == 0 || n_layers == 0) return rc;
  StackGeom g;
  if (!stack_geometry(*s, T, &g)) return AINFER_ERR_SHAPE;
  if (!ws) return AINFER_ERR_NULL;
  if (((uintptr_t)ws) & 255) return AINFER_ERR_WORKSPACE;
  const Layout L = layout_of(*s, 1);
  if (ws_bytes < L.total + (size_t)n_layers * stack_layer_bytes(*s, T, nullptr))
    return AINFER_ERR_WORKSPACE;
  StackWs w;
  w.flags = at<int32_t>(ws, L.stack_flags);
  w.cap = (int)L.stack_cap;
  w.layers = at<uint8_t>(ws, L.total);
  w.err = at<int32_t>(ws, L.sync) + SY_ERR;
  HIP_TRY(launch_decode_stack(s->scale_dtype, *s, g, (const StackLayer *)table, n_layers,
                              resid_in, resid_out, T, norm_mode, eps, w, (hipStream_t)stream));
  return strict_finish(AINFER_OK, ws, stream);
}

int ainfer_moe_route(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *x,
                     int32_t T, int32_t *topk_idx, float *topk_w, float *shared_gate,
                     float *logits, void *ws, size_t ws_bytes, void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (!w || !w->router_w) return AINFER_ERR_NULL;
  if (T == 0) return AINFER_OK;
  if (!x || !topk_idx || !topk_w || !shared_gate) return AINFER_ERR_NULL;
  if ((rc = check_ws(s, chunk_of(T), ws, ws_bytes))) return rc;
  const int H = s->hidden, E = s->n_experts, k = s->top_k;
  for (int t0 = 0; t0 < T; t0 += CHUNK)
    if ((rc = do_route(s, w, (const char *)x + (size_t)t0 * H * 2, chunk_of(T - t0),
                       topk_idx + (size_t)t0 * k, topk_w + (size_t)t0 * k, shared_gate + t0,
                       logits ? logits + (size_t)t0 * E : nullptr, ws, (hipStream_t)stream)))
      return rc;
  return AINFER_OK;
}

int ainfer_moe_experts(const ainfer_moe_shape *s, const ainfer_moe_weights *w, const void *x,
                       const int32_t *topk_idx, int32_t T, void *o, void *ws, size_t ws_bytes,
                       void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (s->precision != AINFER_PRECISION_W4A16) return AINFER_ERR_ARG;
  if (T < 0 || T > AINFER_MOE_CHUNK_TOKENS) return AINFER_ERR_TOKENS;
  if ((rc = check_weights(s, w))) return rc;
  if (T == 0) return AINFER_OK;
  if (!x || !topk_idx || !o) return AINFER_ERR_NULL;
  if ((uintptr_t)x % 16 || (uintptr_t)o % 16) return AINFER_ERR_ARG;
  if ((rc = check_ws(s, T, ws, ws_bytes))) return rc;
  hipStream_t st = (hipStream_t)stream;
  const Layout L = layout_of(*s, T);
  const int H = s->hidden, k = s->top_k, has_shared = s->shared_inter > 0;
  const bool gemm = expert_gemm_at(*s, T);
  DispatchOut d = dispatch_out(s, L, ws, T);
  d.mt = gemm ? gemm_mt(*s, T) : DEC_MT;
  ProfCall pc(st);
  pc.start();
  HIP_TRY(launch_xperm(x, at<uint16_t>(ws, L.xperm), gemm ? at<float>(ws, L.xsum) : nullptr, T,
                       H, st));
  HIP_TRY(launch_dispatch(topk_idx, T, k, s->n_experts, d.mt, has_shared,
                          at<int32_t>(ws, L.chunk_counts), at<int32_t>(ws, L.rank), d, st));
  pc.end(3);
  HIP_TRY_RC(run_experts(s, w, L, ws, d, T, gemm, st, &pc));
  HIP_TRY(launch_gather_rows(at<uint16_t>(ws, L.o), d.inv, o, T, k, H, has_shared, st));
  return AINFER_OK;
}

int ainfer_moe_combine(const ainfer_moe_shape *s, const void *o, const float *topk_w,
                       const float *shared_gate, const void *resid, void *y, int32_t T,
                       void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (T == 0) return AINFER_OK;
  const int has_shared = s->shared_inter > 0;
  if (!o || !topk_w || !y || (has_shared && !shared_gate)) return AINFER_ERR_NULL;
  if ((uintptr_t)o % 16 || (uintptr_t)y % 16 || (resid && (uintptr_t)resid % 16))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_combine((const uint16_t *)o, nullptr, topk_w, shared_gate, has_shared, resid, y,
                         T, s->top_k, s->hidden, nullptr, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_dispatch(const ainfer_moe_shape *s, const int32_t *topk_idx, int32_t T,
                        int32_t *counts, int32_t *offsets, int32_t *perm, int32_t *inv_perm,
                        void *ws, size_t ws_bytes, void *stream) {
  int rc = ainfer_moe_validate(s);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_CHUNK_TOKENS) return AINFER_ERR_TOKENS;
  if (!counts || !offsets) return AINFER_ERR_NULL;
  if (T > 0 && (!topk_idx || !perm)) return AINFER_ERR_NULL;
  if ((rc = check_ws(s, T, ws, ws_bytes))) return rc;
  const Layout L = layout_of(*s, T);
  DispatchOut d;
  memset(&d, 0, sizeof d);
  d.counts = counts;
  d.offsets = offsets;
  d.perm = perm;
  d.inv = inv_perm;
  HIP_TRY(launch_dispatch(topk_idx, T, s->top_k, s->n_experts, DEC_MT, s->shared_inter > 0,
                          at<int32_t>(ws, L.chunk_counts), at<int32_t>(ws, L.rank), d,
                          (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_rmsnorm(const void *x, const void *w, int32_t norm_mode, float eps, void *y,
                       int32_t T, int32_t H, void *stream) {
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (H <= 0 || H % 8) return AINFER_ERR_SHAPE;
  if (norm_mode != AINFER_NORM_PLAIN && norm_mode != AINFER_NORM_ONE_PLUS) return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if (!x || !y) return AINFER_ERR_NULL;
  HIP_TRY(launch_rmsnorm(x, w, norm_mode, eps, y, T, H, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_act_quant_i8(const void *x, int32_t x_dtype, int32_t T, int32_t K, int8_t *q,
                            float *sq, void *stream) {
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (K <= 0 || K % 128) return AINFER_ERR_SHAPE;
  if (x_dtype != AINFER_ACT_F32 && x_dtype != AINFER_ACT_BF16) return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if (!x || !q || !sq) return AINFER_ERR_NULL;
  if ((uintptr_t)x % 8 || (uintptr_t)q % 2 || (uintptr_t)sq % 4) return AINFER_ERR_ARG;
  HIP_TRY(launch_act_quant_i8(x, x_dtype, T, K, q, sq, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_int4_gemv_i8(const uint8_t *packed, const void *scales, int32_t scale_dtype,
                            const int8_t *q, const float *sq, int32_t M, int32_t K, int32_t T,
                            float *y, void *stream) {
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (M <= 0 || K <= 0 || K % 128) return AINFER_ERR_SHAPE;
  if (scale_dtype != AINFER_SCALE_BF16 && scale_dtype != AINFER_SCALE_FP16) return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if (!packed || !scales || !q || !sq || !y) return AINFER_ERR_NULL;
  if ((uintptr_t)packed % 16 || (uintptr_t)q % 16 || (uintptr_t)scales % 2 ||
      (uintptr_t)sq % 4 || (uintptr_t)y % 4)
    return AINFER_ERR_ARG;
  HIP_TRY(launch_int4_gemv_i8(packed, scales, scale_dtype, q, sq, M, K, T, y, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_route_scored(const ainfer_moe_routing *r, const void *logits, int32_t logits_dtype,
                            int64_t ld, const float *bias, int32_t T, int32_t *topk_idx,
                            float *topk_w, void *stream) {
  if (!r) return AINFER_ERR_NULL;
  if (r->n_experts < 1 || r->n_experts > 1024 || r->n_groups < 1 || r->n_groups > 64 ||
      r->n_experts % r->n_groups || r->top_groups < 1 || r->top_groups > r->n_groups)
    return AINFER_ERR_SHAPE;
  if (r->top_k < 1 || r->top_k > 32 ||
      r->top_k > r->top_groups * (r->n_experts / r->n_groups))
    return AINFER_ERR_SHAPE;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if ((r->score != AINFER_SCORE_SOFTMAX && r->score != AINFER_SCORE_SIGMOID) ||
      (r->group_score != AINFER_GROUP_MAX && r->group_score != AINFER_GROUP_TOP2) ||
      (r->renormalize != 0 && r->renormalize != 1) || !std::isfinite(r->scale) || !is_act(logits_dtype))
    return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if (!logits || !topk_idx || !topk_w) return AINFER_ERR_NULL;
  if (ld < r->n_experts || ld > MAX_LD || mis(logits, act_size(logits_dtype)) || mis(bias, 4) ||
      mis(topk_idx, 4) || mis(topk_w, 4))
    return AINFER_ERR_ARG;
  // logits [T][E] may have a pitch, with other rows between theirs; the others are whole
  const size_t out = (size_t)T * r->top_k * 4, all = (size_t)r->n_experts * 4;
  if (meet(topk_idx, out, topk_w, out) || meet(bias, all, topk_idx, out) ||
      meet(bias, all, topk_w, out) || logits == topk_idx || logits == topk_w)
    return AINFER_ERR_ARG;
  HIP_TRY(launch_route_scored(*r, logits, logits_dtype, ld, bias, T, topk_idx, topk_w,
                              (hipStream_t)stream));
  return AINFER_OK;
}

size_t ainfer_moe_lora_workspace_bytes(const ainfer_moe_lora *l, int32_t max_tokens) {
  if (check_lora(l) != AINFER_OK || max_tokens < 0 || max_tokens > AINFER_MOE_MAX_TOKENS) return 0;
  return lora_workspace_bytes(*l, max_tokens > 0 ? max_tokens : 1);
}

int ainfer_moe_lora_apply(const ainfer_moe_lora *l, const void *x, int64_t x_ld,
                          const int32_t *token_adapter, int32_t T, void *const *y,
                          const int64_t *y_ld, void *ws, size_t ws_bytes, void *stream) {
  int rc = check_lora(l);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (T == 0) return AINFER_OK;
  if (!x || !token_adapter || !y || !y_ld || !ws) return AINFER_ERR_NULL;
  for (int p = 0; p < l->n_proj; ++p)
    if (!l->a[p] || !l->b[p] || !y[p]) return AINFER_ERR_NULL;
  const int xsz = act_size(l->x_dtype), ysz = act_size(l->y_dtype);
  if (x_ld < l->in || x_ld > MAX_LD || mis(x, 16) || (x_ld * xsz) % 16 || mis(token_adapter, 4) ||
      mis(l->ranks, 4) || mis(l->scales, 4))
    return AINFER_ERR_ARG;
  for (int p = 0; p < l->n_proj; ++p)
    if (mis(l->a[p], 16) || mis(l->b[p], 16) || mis(y[p], ysz) || y_ld[p] < l->out[p] ||
        y_ld[p] > MAX_LD)
      return AINFER_ERR_ARG;
  if (mis(ws, 256) || ws_bytes < lora_workspace_bytes(*l, T)) return AINFER_ERR_WORKSPACE;
  // what is written (every y, the workspace) at the address of another operand
  auto read = [&](const void *out) {
    bool hit = out == x || out == token_adapter || out == l->ranks || out == l->scales;
    for (int p = 0; p < l->n_proj; ++p) hit |= out == l->a[p] || out == l->b[p];
    return hit;
  };
  if (read(ws)) return AINFER_ERR_ARG;
  for (int p = 0; p < l->n_proj; ++p) {
    if (read(y[p]) || y[p] == ws) return AINFER_ERR_ARG;
    for (int q = 0; q < p; ++q)
      if (y[p] == y[q]) return AINFER_ERR_ARG;
  }
  HIP_TRY(launch_lora(*l, x, x_ld, token_adapter, T, y, y_ld, ws, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_silu_mul(const void *gate, int64_t gate_ld, const void *up, int64_t up_ld,
                        int32_t in_dtype, int32_t T, int32_t I, void *act, int64_t act_ld,
                        int32_t act_dtype, void *stream) {
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (I <= 0) return AINFER_ERR_SHAPE;
  if (!is_act(in_dtype) || !is_act(act_dtype)) return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if (!gate || !up || !act) return AINFER_ERR_NULL;
  const int isz = act_size(in_dtype);
  if (gate_ld < I || up_ld < I || act_ld < I || gate_ld > MAX_LD || up_ld > MAX_LD ||
      act_ld > MAX_LD || mis(gate, isz) || mis(up, isz) || mis(act, act_size(act_dtype)))
    return AINFER_ERR_ARG;
  // in place only where every element of act lies on its own input
  if ((act == gate && (act_dtype != in_dtype || (T > 1 && act_ld != gate_ld))) ||
      (act == up && (act_dtype != in_dtype || (T > 1 && act_ld != up_ld))))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_silu_rows(gate, gate_ld, up, up_ld, in_dtype, T, I, act, act_ld, act_dtype,
                           (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_silu_mul_backward(const void *dact, int64_t dact_ld, const void *gate,
                                 int64_t gate_ld, const void *up, int64_t up_ld, int32_t dtype,
                                 const int32_t *n_live, int32_t N, int32_t I, void *dgate,
                                 int64_t dgate_ld, void *dup, int64_t dup_ld, void *stream) {
  if (N < 0 || N > AINFER_MOE_MAX_ROWS) return AINFER_ERR_TOKENS;
  if (I <= 0 || I > 65536) return AINFER_ERR_SHAPE;
  if (!is_act(dtype)) return AINFER_ERR_ARG;
  if (N == 0) return AINFER_OK;
  if (!dact || !gate || !up || !dgate || !dup) return AINFER_ERR_NULL;
  const int sz = act_size(dtype);
  if (bad_ld(dact_ld, I) || bad_ld(gate_ld, I) || bad_ld(up_ld, I) || bad_ld(dgate_ld, I) ||
      bad_ld(dup_ld, I) || mis(dact, sz) || mis(gate, sz) || mis(up, sz) || mis(dgate, sz) ||
      mis(dup, sz) || mis(n_live, 4))
    return AINFER_ERR_ARG;
  // in place only where every element lies on its own input
  const void *in[3] = {dact, gate, up};
  const int64_t in_ld[3] = {dact_ld, gate_ld, up_ld};
  auto meets = [&](const void *out, int64_t ld, int i) {
    if (out == in[i]) return N > 1 && ld != in_ld[i];
    return over_rows(out, N, ld, I, sz, in[i], N, in_ld[i], I, sz);
  };
  for (int i = 0; i < 3; ++i)
    if (meets(dgate, dgate_ld, i) || meets(dup, dup_ld, i)) return AINFER_ERR_ARG;
  if (over_rows(dgate, N, dgate_ld, I, sz, dup, N, dup_ld, I, sz)) return AINFER_ERR_ARG;
  if (over(dgate, N, dgate_ld, I, sz, n_live, 4) || over(dup, N, dup_ld, I, sz, n_live, 4))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_silu_backward(dact, dact_ld, gate, gate_ld, up, up_ld, dtype, n_live, N, I, dgate,
                               dgate_ld, dup, dup_ld, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_act_quant_fp8(const void *x, int64_t x_ld, int32_t x_dtype, const int32_t *n_live,
                             int32_t N, int32_t K, int32_t scale_kind, uint8_t *q, int64_t q_ld,
                             float *sq, void *stream) {
  if (N < 0 || N > AINFER_MOE_MAX_ROWS) return AINFER_ERR_TOKENS;
  if (K < 16 || K > 65536 || K % 16) return AINFER_ERR_SHAPE;
  if (!is_act(x_dtype) || !is_scale_kind(scale_kind)) return AINFER_ERR_ARG;
  if (N == 0) return AINFER_OK;
  if (!x || !q || !sq) return AINFER_ERR_NULL;
  const int xsz = act_size(x_dtype);
  if (bad_ld(x_ld, K) || bad_ld(q_ld, K) || q_ld % 16 || mis(x, xsz) || mis(q, 16) || mis(sq, 4) ||
      mis(n_live, 4))
    return AINFER_ERR_ARG;
  const size_t scales = (size_t)N * ((K + 127) / 128) * 4;
  if (over_rows(q, N, q_ld, K, 1, x, N, x_ld, K, xsz) || meet(sq, scales, n_live, 4) ||
      over(x, N, x_ld, K, xsz, sq, scales) || over(q, N, q_ld, K, 1, sq, scales) ||
      over(q, N, q_ld, K, 1, n_live, 4))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_act_quant_fp8(x, x_ld, x_dtype, n_live, N, K, scale_kind, q, q_ld, sq,
                               (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_silu_mul_fp8(const void *gate, int64_t gate_ld, const void *up, int64_t up_ld,
                            int32_t in_dtype, const int32_t *n_live, int32_t N, int32_t I,
                            int32_t scale_kind, uint8_t *q, int64_t q_ld, float *sq,
                            void *stream) {
  if (N < 0 || N > AINFER_MOE_MAX_ROWS) return AINFER_ERR_TOKENS;
  if (I < 16 || I > 65536 || I % 16) return AINFER_ERR_SHAPE;
  if (!is_act(in_dtype) || !is_scale_kind(scale_kind)) return AINFER_ERR_ARG;
  if (N == 0) return AINFER_OK;
  if (!gate || !up || !q || !sq) return AINFER_ERR_NULL;
  const int sz = act_size(in_dtype);
  if (bad_ld(gate_ld, I) || bad_ld(up_ld, I) || bad_ld(q_ld, I) || q_ld % 16 || mis(gate, sz) ||
      mis(up, sz) || mis(q, 16) || mis(sq, 4) || mis(n_live, 4))
    return AINFER_ERR_ARG;
  const size_t scales = (size_t)N * ((I + 127) / 128) * 4;
  if (over_rows(q, N, q_ld, I, 1, gate, N, gate_ld, I, sz) ||
      over_rows(q, N, q_ld, I, 1, up, N, up_ld, I, sz) || meet(sq, scales, n_live, 4) ||
      over(gate, N, gate_ld, I, sz, sq, scales) ||
      over(up, N, up_ld, I, sz, sq, scales) || over(q, N, q_ld, I, 1, sq, scales) ||
      over(q, N, q_ld, I, 1, n_live, 4))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_silu_mul_fp8(gate, gate_ld, up, up_ld, in_dtype, n_live, N, I, scale_kind, q, q_ld,
                              sq, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_weight_quant_fp8(const void *w, int32_t w_dtype, int32_t E, int32_t M, int32_t K,
                                int32_t scale_kind, uint8_t *q, float *scales, void *stream) {
  int rc = check_fp8_sizes(E, M, K);
  if (rc) return rc;
  if (!is_act(w_dtype) || !is_scale_kind(scale_kind)) return AINFER_ERR_ARG;
  if (!w || !q || !scales) return AINFER_ERR_NULL;
  if (mis(w, act_size(w_dtype)) || mis(q, 16) || mis(scales, 4)) return AINFER_ERR_ARG;
  const size_t n = (size_t)E * M * K, sn = (size_t)E * ((M + 127) / 128) * ((K + 127) / 128) * 4;
  if (meet(w, n * act_size(w_dtype), q, n) || meet(w, n * act_size(w_dtype), scales, sn) ||
      meet(q, n, scales, sn))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_weight_quant_fp8(w, w_dtype, E, M, K, scale_kind, q, scales, (hipStream_t)stream));
  return AINFER_OK;
}

size_t ainfer_moe_fp8_packed_bytes(int32_t E, int32_t M, int32_t K) {
  return check_fp8_sizes(E, M, K) == AINFER_OK ? fp8_packed_bytes(E, M, K) : 0;
}

int ainfer_moe_fp8_pack(const uint8_t *w, int32_t E, int32_t M, int32_t K, int32_t transpose,
                        uint8_t *packed, size_t packed_bytes, void *stream) {
  int rc = check_fp8_sizes(E, M, K);
  if (rc) return rc;
  if (transpose != 0 && transpose != 1) return AINFER_ERR_ARG;
  if (!w || !packed) return AINFER_ERR_NULL;
  const size_t n = fp8_packed_bytes(E, M, K);
  if (mis(packed, 16) || (!transpose && mis(w, 16)) || packed_bytes < n ||
      meet(w, (size_t)E * M * K, packed, n))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_fp8_pack(w, E, M, K, transpose, packed, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_fp8_product(const ainfer_moe_fp8 *w, const uint8_t *q, int64_t q_ld, const float *sq,
                           const int32_t *offsets, int32_t N, void *y, int64_t y_ld,
                           void *stream) {
  int rc = check_fp8(w);
  if (rc) return rc;
  if (N < 0 || N > AINFER_MOE_MAX_ROWS) return AINFER_ERR_TOKENS;
  if (N == 0) return AINFER_OK;
  if (!w->packed || !w->scales || !q || !sq || !y || (!offsets && w->n_experts != 1))
    return AINFER_ERR_NULL;
  const int M = w->rows, K = w->cols, ysz = act_size(w->y_dtype);
  // a tile's rows of codes are addressed with 32-bit offsets
  if (bad_ld(q_ld, K) || q_ld % 16 || q_ld > 1 << 24 || bad_ld(y_ld, M) || mis(w->packed, 16) ||
      mis(q, 16) || mis(w->scales, 4) || mis(sq, 4) || mis(offsets, 4) || mis(y, ysz))
    return AINFER_ERR_ARG;
  const size_t G = (K + 127) / 128, E = w->n_experts;
  if (over(y, N, y_ld, M, ysz, w->packed, fp8_packed_bytes(w->n_experts, M, K)) ||
      over(y, N, y_ld, M, ysz, w->scales, E * ((M + 127) / 128) * G * 4) ||
      over(y, N, y_ld, M, ysz, sq, N * G * 4) || over(y, N, y_ld, M, ysz, offsets, (E + 1) * 4) ||
      over_rows(y, N, y_ld, M, ysz, q, N, q_ld, K, 1))
    return AINFER_ERR_ARG;
  const Fp8Args a = {w->packed, w->scales, q, sq, offsets, y, q_ld, y_ld, w->n_experts, M, K, N};
  HIP_TRY(launch_fp8_product(a, w->y_dtype, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_debug_fp8_form(int32_t E, int32_t M, int32_t K, int32_t N, int32_t y_dtype,
                              int32_t *weight_rows, int32_t *rows) {
  int rc = check_fp8_sizes(E, M, K);
  if (rc) return rc;
  if (N < 1 || N > AINFER_MOE_MAX_ROWS) return AINFER_ERR_TOKENS;
  if (!is_act(y_dtype)) return AINFER_ERR_ARG;
  if (!weight_rows || !rows) return AINFER_ERR_NULL;
  const Fp8Form form = fp8_form(E, M, K, N, y_dtype == AINFER_ACT_F32);
  *weight_rows = form.m;
  *rows = form.rows;
  return AINFER_OK;
}

size_t ainfer_moe_sort_workspace_bytes(int32_t max_tokens, int32_t top_k, int32_t n_experts) {
  if (max_tokens < 0 || max_tokens > AINFER_MOE_MAX_TOKENS || top_k < 1 || top_k > 32 ||
      n_experts < 1 || n_experts > 1024)
    return 0;
  return sort_workspace_bytes(max_tokens > 0 ? max_tokens : 1, top_k, n_experts);
}

int ainfer_moe_sort_rows(const ainfer_moe_sorting *s, const void *x, int64_t x_ld,
                         const int32_t *topk_idx, int32_t T, int32_t *offsets, int32_t *pos,
                         void *rows, int64_t rows_ld, float *row_scales, void *ws, size_t ws_bytes,
                         void *stream) {
  int rc = check_sorting(s);
  if (rc) return rc;
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS) return AINFER_ERR_TOKENS;
  if (!offsets) return AINFER_ERR_NULL;
  if (mis(offsets, 4)) return AINFER_ERR_ARG;
  const int k = s->top_k, H = s->hidden, xsz = act_size(s->x_dtype), rsz = s->fp8 ? 1 : xsz;
  const int64_t P = (int64_t)T * k;
  const size_t n = (size_t)P * 4, no = ((size_t)s->n_experts + 1) * 4,
               ns = (size_t)P * ((H + 127) / 128) * 4;
  if (T > 0) {
    if (!topk_idx || !pos || !ws || (rows && (!x || (s->fp8 && !row_scales))))
      return AINFER_ERR_NULL;
    if (mis(topk_idx, 4) || mis(pos, 4)) return AINFER_ERR_ARG;
    if (rows && (bad_ld(x_ld, H) || bad_ld(rows_ld, H) || mis(x, xsz) ||
                 (s->fp8 && (rows_ld % 16 || mis(rows, 16) || mis(row_scales, 4))) || mis(rows, rsz)))
      return AINFER_ERR_ARG;
    if (mis(ws, 256) || ws_bytes < sort_workspace_bytes(T, k, s->n_experts))
      return AINFER_ERR_WORKSPACE;
    // what is written (offsets, pos, the workspace, rows, their scales) over another operand
    const size_t nw = sort_workspace_bytes(T, k, s->n_experts);
    float *sc = rows && s->fp8 ? row_scales : nullptr;
    if (meet(offsets, no, pos, n) || meet(offsets, no, topk_idx, n) || meet(pos, n, topk_idx, n) ||
        meet(ws, nw, offsets, no) || meet(ws, nw, pos, n) || meet(ws, nw, topk_idx, n) ||
        meet(sc, ns, offsets, no) || meet(sc, ns, pos, n) || meet(sc, ns, topk_idx, n) ||
        meet(sc, ns, ws, nw))
      return AINFER_ERR_ARG;
    if (rows) {
      auto hit = [&](const void *p, size_t bytes) {
        return over(rows, P, rows_ld, H, rsz, p, bytes) || over(x, T, x_ld, H, xsz, p, bytes);
      };
      if (over_rows(rows, P, rows_ld, H, rsz, x, T, x_ld, H, xsz) || hit(offsets, no) ||
          hit(pos, n) || hit(ws, nw) || hit(sc, ns) ||
          over(rows, P, rows_ld, H, rsz, topk_idx, n))
        return AINFER_ERR_ARG;
    }
  }
  HIP_TRY(launch_sort_rows(*s, x, x_ld, topk_idx, T, offsets, pos, T > 0 ? rows : nullptr, rows_ld,
                           row_scales, ws, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_unpermute(const void *rows, int64_t rows_ld, int32_t rows_dtype, int32_t N,
                         const int32_t *pos, const float *w, int32_t T, int32_t top_k, int32_t H,
                         const void *resid, int64_t resid_ld, void *y, int64_t y_ld,
                         int32_t y_dtype, void *stream) {
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS || N < 0 || N > AINFER_MOE_MAX_ROWS)
    return AINFER_ERR_TOKENS;
  if (top_k < 1 || top_k > 32 || H < 1 || H > 65536) return AINFER_ERR_SHAPE;
  if (!is_act(rows_dtype) || !is_act(y_dtype)) return AINFER_ERR_ARG;
  if (T == 0) return AINFER_OK;
  if ((!rows && N > 0) || !pos || !y) return AINFER_ERR_NULL;
  const int rsz = act_size(rows_dtype), ysz = act_size(y_dtype);
  if (bad_ld(rows_ld, H) || bad_ld(y_ld, H) || (resid && bad_ld(resid_ld, H)) || mis(rows, rsz) ||
      mis(pos, 4) || mis(w, 4) || mis(resid, ysz) || mis(y, ysz))
    return AINFER_ERR_ARG;
  const size_t n = (size_t)T * top_k * 4;
  if (over_rows(y, T, y_ld, H, ysz, rows, N, rows_ld, H, rsz) ||
      over(y, T, y_ld, H, ysz, pos, n) || over(y, T, y_ld, H, ysz, w, n) ||
      (resid == y ? T > 1 && resid_ld != y_ld
                  : over_rows(y, T, y_ld, H, ysz, resid, T, resid_ld, H, ysz)))
    return AINFER_ERR_ARG;
  HIP_TRY(launch_unpermute(rows, rows_ld, rows_dtype, N, pos, w, T, top_k, H, resid, resid_ld, y,
                           y_ld, y_dtype, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_unpermute_backward(const void *dy, int64_t dy_ld, int32_t dy_dtype, const void *rows,
                                  int64_t rows_ld, int32_t rows_dtype, int32_t N,
                                  const int32_t *pos, const float *w, int32_t T, int32_t top_k,
                                  int32_t H, void *drows, int64_t drows_ld, float *dw,
                                  void *stream) {
  if (T < 0 || T > AINFER_MOE_MAX_TOKENS || N < 0 || N > AINFER_MOE_MAX_ROWS)
    return AINFER_ERR_TOKENS;
  if (top_k < 1 || top_k > 32 || H < 1 || H > 65536) return AINFER_ERR_SHAPE;
  if (!is_act(rows_dtype) || !is_act(dy_dtype)) return AINFER_ERR_ARG;
  if (T == 0 || (!drows && !dw)) return AINFER_OK;
  if (!dy || !pos || (dw && !rows && N > 0)) return AINFER_ERR_NULL;
  const int rsz = act_size(rows_dtype), ysz = act_size(dy_dtype);
  if (bad_ld(dy_ld, H) || (dw && bad_ld(rows_ld, H)) || (drows && bad_ld(drows_ld, H)) ||
      mis(dy, ysz) || mis(rows, rsz) || mis(drows, rsz) || mis(pos, 4) || mis(w, 4) || mis(dw, 4))
    return AINFER_ERR_ARG;
  const size_t n = (size_t)T * top_k * 4;
  if (meet(dw, n, pos, n) || meet(dw, n, w, n) || over(dy, T, dy_ld, H, ysz, dw, n) ||
      (dw && N > 0 && over(rows, N, rows_ld, H, rsz, dw, n)) || (drows && drows == dy))
    return AINFER_ERR_ARG;
  if (drows && N > 0) {
    if (over(drows, N, drows_ld, H, rsz, pos, n) || over(drows, N, drows_ld, H, rsz, w, n) ||
        over(drows, N, drows_ld, H, rsz, dw, n) ||
        over_rows(drows, N, drows_ld, H, rsz, dy, T, dy_ld, H, ysz) ||
        (dw && over_rows(drows, N, drows_ld, H, rsz, rows, N, rows_ld, H, rsz)))
      return AINFER_ERR_ARG;
  }
  HIP_TRY(launch_unpermute_backward(dy, dy_ld, dy_dtype, rows, rows_ld, rows_dtype, N, pos, w, T,
                                    top_k, H, drows, drows_ld, dw, (hipStream_t)stream));
  return AINFER_OK;
}

int ainfer_moe_profile_enable(int32_t enable) {
  if (enable && !g_prof.created) {
    for (int i = 0; i < PROF_SLOTS; ++i)
      for (int j = 0; j <= NSTAGE; ++j) {
        if (hipEventCreate(&g_prof.ev[i][j]) != hipSuccess) return AINFER_ERR_HIP;
        g_prof.used[i][j] = false;
      }
    for (int i = 0; i < PROF_SLOTS; ++i) {
      for (int j = 0; j < 2; ++j)
        if (hipEventCreate(&g_prof.kev[i][j]) != hipSuccess) return AINFER_ERR_HIP;
      g_prof.kused[i] = false;
    }
    g_prof.created = true;
  }
  if (enable) {
    for (int i = 0; i < NSTAGE; ++i) g_prof.sum_us[i] = 0.0, g_prof.cnt[i] = 0;
    g_prof.calls = 0;
    g_prof.slot = 0;
    g_prof.ksum_us = 0.0;
    g_prof.kcnt = 0;
    if (g_prof.created)
      for (int i = 0; i < PROF_SLOTS; ++i) {
        for (int j = 0; j <= NSTAGE; ++j) g_prof.used[i][j] = false;
        g_prof.kused[i] = false;
      }
  }
  g_prof.on = enable != 0;
  return AINFER_OK;
}

int ainfer_moe_profile_read(float *stage_us, int32_t n_stages, int32_t *n_calls) {
  if (!stage_us && n_stages > 0) return AINFER_ERR_NULL;
  if (g_prof.created)
    for (int i = 0; i < PROF_SLOTS; ++i) prof_flush_slot(i);
  for (int i = 0; i < n_stages && i < NSTAGE; ++i)
    stage_us[i] = g_prof.cnt[i] ? (float)(g_prof.sum_us[i] / g_prof.cnt[i]) : 0.0f;
  if (n_calls) *n_calls = g_prof.calls;
  return AINFER_OK;
}

int ainfer_moe_profile_kernel(float *gate_up_us, int32_t *n_launches) {
  if (!gate_up_us) return AINFER_ERR_NULL;
  if (g_prof.created)
    for (int i = 0; i < PROF_SLOTS; ++i) prof_flush_slot(i);
  *gate_up_us = g_prof.kcnt ? (float)(g_prof.ksum_us / g_prof.kcnt) : 0.0f;
  if (n_launches) *n_launches = g_prof.kcnt;
  return AINFER_OK;
}

int ainfer_moe_debug_spin_limit(int32_t polls) {
  if (polls < 0) return AINFER_ERR_ARG;
  g_spin_max = polls;
  return AINFER_OK;
}

int ainfer_moe_fill(int32_t kind, uint64_t seed, float std_, size_t n, void *out,
                    void *stream) {
  if (kind < AINFER_FILL_BYTES || kind > AINFER_FILL_BF16_ABSNORMAL) return AINFER_ERR_ARG;
  if (n == 0) return AINFER_OK;
  if (!out) return AINFER_ERR_NULL;
  HIP_TRY(launch_fill(kind, seed, std_, n, out, (hipStream_t)stream));
  return AINFER_OK;
}

}  // extern "C"
