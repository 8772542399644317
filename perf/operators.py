"""The operators around the expert stage that a served model adds, measured.

Three kinds of call:

  route  scored routing: softmax or sigmoid scores of given logits, a selection
         bias, expert groups, top-k, weights renormalised and scaled
  lora   low-rank adapters of many requests beside one to four shared
         projections of the same input: y_p += scale_a * (x A_a^T) B_a^T
  silu   the gated activation between an MLP's projections

over single decode steps, batched decode, ragged and full prefill chunks and
the largest call the library takes.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _route(name, tokens, experts, top_k, score="sigmoid", bias=True, groups=1, top_groups=1,
           group_score="top2", renorm=True, dtype="fp32"):
    return dict(name=name, op="route", tokens=tokens, experts=experts, top_k=top_k, score=score,
                bias=bias, groups=groups, top_groups=top_groups, group_score=group_score,
                renorm=renorm, dtype=dtype)


def _lora(name, tokens, requests, adapters, rank, cols, rows, projs=1, x="bf16", y="bf16",
          ragged=False):
    return dict(name=name, op="lora", tokens=tokens, requests=requests, adapters=adapters,
                rank=rank, cols=cols, rows=rows, projs=projs, x=x, y=y, ragged=ragged)


def _silu(name, tokens, inter, x, y):
    return dict(name=name, op="silu", tokens=tokens, inter=inter, x=x, y=y)


def listed():
    return [
        # one decode step's token: grouped sigmoid routing with a balance bias (all latency)
        _route("route_T1_E256_groups", 1, 256, 8, groups=8, top_groups=4),
        # a ragged decode batch: an odd expert count, groups by their best expert, bf16 logits
        _route("route_T333_E60_softmax", 333, 60, 4, score="softmax", bias=False, groups=6,
               top_groups=3, group_score="max", renorm=False, dtype="bf16"),
        # a full prefill chunk, grouped sigmoid routing
        _route("route_T4096_E256_groups", 4096, 256, 8, groups=8, top_groups=4),
        # the largest call of the library: biased softmax over the benchmark's 512 experts
        _route("route_T65536_E512_bias", 65536, 512, 10, score="softmax"),
        # one token of one request: an attention-sized projection (all latency)
        _lora("lora_T1_K4096", 1, 1, 32, 16, 4096, 4096),
        # batched decode, every sequence its own adapter: the shared expert's gate and up in fp32
        _lora("lora_T64_gate_up", 64, 64, 64, 16, 4096, 1024, projs=2, y="fp32", ragged=True),
        # batched decode of a large dense MLP projection with high-rank adapters
        _lora("lora_T16_K5120", 16, 16, 16, 64, 5120, 17408, y="fp32"),
        # ragged prompts of seven requests: the shared expert's down from fp32 act rows
        _lora("lora_T1003_down", 1003, 7, 12, 8, 1024, 4096, x="fp32", y="fp32"),
        # a full prefill chunk of ragged prompts
        _lora("lora_T4096_K4096", 4096, 24, 64, 32, 4096, 4096),
        # batched decode of the shared expert in the W4A8 precision
        _silu("silu_T16_I1024", 16, 1024, "fp32", "fp32"),
        # a full prefill chunk of a large dense MLP
        _silu("silu_T4096_I17408", 4096, 17408, "bf16", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("route", "route", "lora", "lora", "lora", "silu"))
        if kind == "route":
            groups = rng.choice((1, 1, 2, 3, 4, 8, 8, 16))
            per = _log_int(rng, 8, 512) if groups == 1 else _log_int(rng, 4, 1024 // groups)
            top_groups = rng.randint(1, groups)
            c = _route("", _log_int(rng, 1, 65536), groups * per, 1, rng.choice(("softmax", "sigmoid")),
                       rng.random() < 0.7, groups, top_groups, rng.choice(("max", "top2")),
                       rng.random() < 0.7, rng.choice(("fp32", "fp32", "bf16")))
            c["top_k"] = rng.randint(1, min(16, top_groups * per))
        elif kind == "lora":
            tokens = _log_int(rng, 1, 8192)
            adapters = _log_int(rng, 1, 128)
            requests = min(tokens, _log_int(rng, 1, 96)) if tokens > 96 else tokens
            c = _lora("", tokens, requests, adapters, 8 * _log_int(rng, 1, 16),
                      8 * _log_int(rng, 32, 1024), _log_int(rng, 200, 8192),
                      rng.choice((1, 1, 2, 3)), rng.choice(("bf16", "bf16", "fp32")),
                      rng.choice(("bf16", "fp32")), rng.random() < 0.5)
        else:
            c = _silu("", _log_int(rng, 1, 8192), _log_int(rng, 100, 17408),
                      *rng.choice((("fp32", "fp32"), ("bf16", "bf16"), ("fp32", "bf16"))))
        if _cost(c) <= most and _state_bytes(c) < 4 << 30:
            del c["name"]
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _state_bytes(case):
    if case["op"] != "lora":
        return work(case)["bytes"]
    per = case["rank"] * (case["cols"] + case["rows"]) * case["projs"]
    # the plain form's 32-bit weights of every adapter, or of every token
    return 2 * per * case["adapters"] + 8 * per * min(case["adapters"], case["tokens"])


def _used(case):
    """Requests with an adapter, and the adapters they use at most."""
    n = case["requests"]
    with_one = n - (n // 8)
    return with_one, min(with_one, case["adapters"])


def _size(dtype):
    return 4 if dtype == "fp32" else 2


def work(case):
    T = case["tokens"]
    if case["op"] == "route":
        E = case["experts"]
        b = T * E * _size(case["dtype"]) + T * case["top_k"] * 8 + (4 * E if case["bias"] else 0)
        return {"bytes": b, "flops": 10 * T * E}
    if case["op"] == "silu":
        n = T * case["inter"]
        return {"bytes": n * (2 * _size(case["x"]) + _size(case["y"])), "flops": 8 * n}
    R, K, M, P = case["rank"], case["cols"], case["rows"], case["projs"]
    if case["ragged"]:
        R = (R + 1) / 2
    with_one, used = _used(case)
    rows = T * with_one / case["requests"]
    b = rows * (K * _size(case["x"]) + 2 * P * M * _size(case["y"])) + 2 * used * R * P * (K + M)
    return {"bytes": b, "flops": 2 * rows * R * P * (K + M)}


# ---- inputs -------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)

    T = case["tokens"]
    s = dict(case=case)
    if case["op"] == "route":
        E = case["experts"]
        s["logits"] = normal(T, E, std=1.5, dtype=DT[case["dtype"]])
        s["bias"] = None
        if case["bias"]:
            s["bias"] = normal(E, std=0.1 if case["score"] == "sigmoid" else 1.0 / E)
        # what a serving program keeps: the routing description and the output rows
        s["idx"] = torch.empty(T, case["top_k"], dtype=torch.int32, device=DEV)
        s["w"] = torch.empty(T, case["top_k"], dtype=torch.float32, device=DEV)
        if own:
            from ainfer_amd import _lib as L
            s["routing"] = L.Routing(
                E, case["top_k"],
                L.SCORE_SOFTMAX if case["score"] == "softmax" else L.SCORE_SIGMOID,
                case["groups"], case["top_groups"],
                L.GROUP_MAX if case["group_score"] == "max" else L.GROUP_TOP2,
                int(case["renorm"]), SCALE)
    elif case["op"] == "silu":
        s["g"] = normal(T, case["inter"], std=2.0, dtype=DT[case["x"]])
        s["u"] = normal(T, case["inter"], dtype=DT[case["x"]])
        s["act"] = torch.empty(T, case["inter"], dtype=DT[case["y"]], device=DEV)
    else:
        R, K, M, P, N = (case[n] for n in ("rank", "cols", "rows", "projs", "adapters"))
        s["x"] = normal(T, K, dtype=DT[case["x"]])
        s["a"] = [normal(N, R, K, std=K ** -0.5, dtype=torch.bfloat16) for _ in range(P)]
        s["b"] = [normal(N, M, R, std=0.1, dtype=torch.bfloat16) for _ in range(P)]
        s["y"] = [normal(T, M, dtype=DT[case["y"]]) for _ in range(P)]
        s["scales"] = torch.rand(N, generator=g, device=DEV) + 0.5
        s["ranks"] = None
        if case["ragged"]:
            s["ranks"] = torch.randint(1, R + 1, (N,), generator=g, device=DEV, dtype=torch.int32)
        s["ids"] = _token_adapters(case, g)
        if own:
            from ainfer_amd.moe import LoraAdapters
            s["lora"] = LoraAdapters(s["a"], s["b"], ranks=s["ranks"], scales=s["scales"],
                                     x_dtype=DT[case["x"]], y_dtype=DT[case["y"]])
            s["ws"] = s["lora"].workspace(T)
    return s


SCALE = 2.5  # what the routed weights are multiplied by


def _token_adapters(case, g):
    """token -> adapter: requests of random lengths one after the other, each
    with an adapter of its own while they last, every eighth without one."""
    T, n, N = case["tokens"], case["requests"], case["adapters"]
    if n == T:
        request = torch.arange(T, device=DEV)
    else:
        cuts = torch.randperm(T - 1, generator=g, device=DEV)[:n - 1] + 1
        request = torch.zeros(T, dtype=torch.int64, device=DEV)
        request[cuts] = 1
        request = request.cumsum(0)
    of_request = torch.randperm(max(n, N), generator=g, device=DEV)[:n] % N
    at = torch.arange(n, device=DEV)
    of_request = torch.where(at % 8 == 7, torch.full_like(of_request, -1), of_request)
    return of_request[request].to(torch.int32)


# ---- one pass -------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        from ainfer_amd import moe
        if case["op"] == "route":
            moe.route_scored(s["routing"], s["logits"], s["bias"], out=(s["idx"], s["w"]))
            return s["idx"], s["w"]
        if case["op"] == "silu":
            moe.silu_mul(s["g"], s["u"], s["act"])
            return s["act"]
        s["lora"].apply(s["x"], s["ids"], s["y"], s["ws"])
        return s["y"]
    if case["op"] == "route":
        return _plain_route(s)
    if case["op"] == "silu":
        g, u = s["g"].float(), s["u"].float()
        s["act"].copy_(g / (1 + torch.exp(-g)) * u)
        return s["act"]
    return _plain_lora(s)


def _plain_route(s):
    # in 64 bits: two experts' scores can be nearer than 32 bits tell apart
    case = s["case"]
    T, E, G = case["tokens"], case["experts"], case["groups"]
    logits = s["logits"].double()
    if case["score"] == "softmax":
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    biased = score if s["bias"] is None else score + s["bias"].double()
    key = logits if s["bias"] is None else biased
    if G > 1:
        if case["group_score"] == "max":
            best = key.view(T, G, E // G).amax(2)
        else:
            best = biased.view(T, G, E // G).sort(dim=2, descending=True)[0][:, :, :2].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        left_out = torch.ones(T, G, dtype=torch.bool, device=DEV).scatter_(1, kept, False)
        key = key.masked_fill(left_out.repeat_interleave(E // G, 1), -math.inf)
    idx = key.sort(dim=1, descending=True, stable=True)[1][:, :case["top_k"]]
    w = score.gather(1, idx)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    s["idx"].copy_(idx)
    s["w"].copy_(w * SCALE)
    return s["idx"], s["w"]


def _plain_lora(s):
    case = s["case"]
    R, N = case["rank"], case["adapters"]
    ids = s["ids"].long()
    has = ids >= 0
    ids = ids.clamp_min(0)
    scale = s["scales"][ids] * has
    rank = torch.full_like(ids, R) if s["ranks"] is None else s["ranks"].long()[ids]
    x = s["x"].float()
    live = torch.arange(R, device=DEV)[None, :] < rank[:, None]
    v = [_down(x, a, ids, live, scale, N) for a in s["a"]]
    delta = [_up(p, b, ids, N) for p, b in zip(v, s["b"])]
    y = [o + d for o, d in zip(s["y"], delta)]
    torch._foreach_copy_(s["y"], y)
    return s["y"]


def _down(x, a, ids, live, scale, N):
    """[T][R]: each token through its own adapter's A.  Few tokens take their
    adapters' weights one by one, many tokens a product with every adapter's."""
    T, R = live.shape
    if T <= N:
        v = (a[ids].float() * x[:, None, :]).sum(2)
    else:
        v = (x @ a.float().flatten(0, 1).t()).view(T, N, R)[torch.arange(T, device=DEV), ids]
    return v * live * scale[:, None]


def _up(v, b, ids, N):
    T, R = v.shape
    if T <= N:
        return (b[ids].float() * v[:, None, :]).sum(2)
    wide = torch.zeros(T, N, R, device=DEV)
    wide[torch.arange(T, device=DEV), ids] = v
    return wide.flatten(1) @ b.float().transpose(1, 2).reshape(N * R, -1)


# ---- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "silu":
        g, u = s["g"].double(), s["u"].double()
        return u * g * torch.sigmoid(g)
    if case["op"] == "route":
        return _exact_route(case, s["logits"].double(), s["bias"])
    out = [y.double() for y in s["y"]]
    ids = s["ids"].tolist()
    for n in sorted(set(ids) - {-1}):
        rows = torch.tensor([t for t, i in enumerate(ids) if i == n], device=DEV)
        r = case["rank"] if s["ranks"] is None else int(s["ranks"][n])
        for y, a, b in zip(out, s["a"], s["b"]):
            low = s["x"][rows].double() @ a[n, :r].double().t().contiguous()
            y[rows] += float(s["scales"][n]) * (low @ b[n, :, :r].double().t().contiguous())
    return out


def _exact_route(case, logits, bias):
    T, E, G = case["tokens"], case["experts"], case["groups"]
    score = torch.softmax(logits, 1) if case["score"] == "softmax" else torch.sigmoid(logits)
    shifted = score + (0 if bias is None else bias.double())
    order = shifted.clone() if bias is not None else logits.clone()
    if G > 1:
        by_group = shifted.view(T, G, -1)
        if case["group_score"] == "max":
            value = order.view(T, G, -1).max(2).values
        else:
            value = by_group.topk(min(2, E // G), 2).values.sum(2)
        # a group stays while fewer than top_groups are better, or equal and before it
        ahead = (value[:, None, :] > value[:, :, None]) | (
            (value[:, None, :] == value[:, :, None])
            & torch.ones(G, G, dtype=torch.bool, device=DEV).tril(-1))
        stays = ahead.sum(2) < case["top_groups"]
        order = torch.where(stays[:, :, None], order.view(T, G, -1),
                            torch.full((), -math.inf, dtype=torch.float64, device=DEV)).view(T, E)
    idx, w = [], []
    at = torch.arange(E, device=DEV)
    for _ in range(case["top_k"]):
        best = order.max(1, keepdim=True).values
        pick = torch.where(order == best, at, E).min(1).values
        idx.append(pick)
        w.append(score.gather(1, pick[:, None])[:, 0])
        order.scatter_(1, pick[:, None], -math.inf)
    w = torch.stack(w, 1)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return torch.stack(idx, 1).to(torch.int32), w * SCALE
