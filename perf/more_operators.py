"""The operators of an expert stage in 8-bit floating point, measured.

Four kinds of call:

  product  y = x W^T with e4m3 codes on both sides, a scale for every 128 columns
           of x and for every 128 x 128 block of W, rows sorted by expert (or one
           matrix for all)
  sort     token rows copied into expert order, as they are or quantised to e4m3,
           from the router's ids; ids of experts that live elsewhere are dropped
  back     the experts' rows weighted and summed per token, and its gradient
  act      the gated activation written as e4m3 codes and scales, and its gradient

over single decode steps, batched decode, ragged and full prefill chunks, and
training steps.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
TOP = 448.0     # the largest e4m3 value
LEAST = 2.0 ** -126


def _product(name, tokens, experts, top_k, rows, cols, y="bf16", local=1.0):
    return dict(name=name, op="product", tokens=tokens, experts=experts, top_k=top_k, rows=rows,
                cols=cols, y=y, local=local)


def _sort(name, tokens, experts, top_k, hidden, x="bf16", to="fp8", pow2=False, elsewhere=0):
    return dict(name=name, op="sort", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden,
                x=x, to=to, pow2=pow2, elsewhere=elsewhere)


def _back(name, tokens, experts, top_k, hidden, grad=False, rows="bf16", y="bf16", resid=False,
          elsewhere=0):
    return dict(name=name, op="back", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden,
                grad=grad, rows=rows, y=y, resid=resid, elsewhere=elsewhere)


def _act(name, rows, inter, grad=False, x="bf16", pow2=False):
    return dict(name=name, op="act", rows=rows, inter=inter, grad=grad, x=x, pow2=pow2)


def listed():
    return [
        # one decode step of a dense projection: 89 MB of weights for one row
        _product("product_T1_M17408_K5120", 1, 1, 1, 17408, 5120),
        # batched decode: 128 rows spread over 256 experts' gate and up
        _product("product_T16_E256", 16, 256, 8, 1024, 2048),
        # ragged prompts where a third of the pairs belong to other GPUs' experts, fp32 rows
        _product("product_T1003_E96", 1003, 96, 6, 1792, 2560, y="fp32", local=0.66),
        # a full prefill chunk: gate and up of 64 experts
        _product("product_T4096_E64", 4096, 64, 8, 2048, 4096),
        # one decode step's token, quantised for its eight experts (all latency)
        _sort("sort_T1_fp8", 1, 256, 8, 4096),
        # a full prefill chunk over the benchmark's 512 experts, power-of-two scales
        _sort("sort_T4096_fp8", 4096, 512, 10, 2048, pow2=True),
        # two chunks of a training step, rows as they are; half of the experts elsewhere
        _sort("sort_T8192_bf16", 8192, 64, 8, 4096, to="bf16", elsewhere=64),
        # batched decode: expert rows and the residual stream
        _back("back_T16", 16, 256, 8, 2048, resid=True),
        # a full prefill chunk
        _back("back_T4096", 4096, 512, 10, 2048),
        # a training step's chunk: the rows' and the routing weights' gradients
        _back("back_grad_T4096", 4096, 64, 8, 4096, grad=True),
        # batched decode: 128 expert rows
        _act("act_R128", 128, 512),
        # a training step's chunk: gradients of gate and up
        _act("act_grad_R32768", 32768, 1024, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("product", "product", "product", "sort", "sort", "back", "back", "act"))
        experts = _log_int(rng, 2, 512)
        top_k = rng.randint(1, min(10, experts))
        tokens = _log_int(rng, 1, 8192)
        if kind == "product":
            if rng.random() < 0.3:
                experts = top_k = 1
            c = _product("", tokens, experts, top_k, _log_int(rng, 130, 17408),
                         16 * _log_int(rng, 16, 512), rng.choice(("bf16", "fp32")),
                         rng.choice((1.0, 1.0, 0.5)))
        elif kind == "sort":
            x = rng.choice(("bf16", "bf16", "fp32"))
            c = _sort("", tokens, experts, top_k, 16 * _log_int(rng, 16, 512), x,
                      rng.choice(("fp8", "fp8", x)), rng.random() < 0.5,
                      rng.choice((0, 0, experts)))
            c["pow2"] = c["pow2"] and c["to"] == "fp8"
        elif kind == "back":
            c = _back("", tokens, experts, top_k, _log_int(rng, 200, 8192), rng.random() < 0.5,
                      rng.choice(("bf16", "bf16", "fp32")), rng.choice(("bf16", "fp32")),
                      rng.random() < 0.5, rng.choice((0, 0, experts)))
            c["resid"] = c["resid"] and not c["grad"]
        else:
            c = _act("", _log_int(rng, 1, 65536), 16 * _log_int(rng, 8, 512), rng.random() < 0.5,
                     rng.choice(("bf16", "bf16", "fp32")), rng.random() < 0.5)
            c["pow2"] = c["pow2"] and not c["grad"]
        if _cost(c) <= most and _state_bytes(c) < 1 << 30:
            del c["name"]
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200)


def _state_bytes(case):
    if case["op"] == "product":
        return case["experts"] * case["rows"] * case["cols"] + work(case)["bytes"]
    return work(case)["bytes"]


def _size(dtype):
    return {"fp32": 4, "bf16": 2, "fp8": 1}[dtype]


def _groups(n):
    return -(-n // 128)


def _kept(case):
    """Pairs of a token and an expert that stay here, about."""
    n = case["tokens"] * case["top_k"]
    return n * case["experts"] / (case["experts"] + case["elsewhere"])


def work(case):
    if case["op"] == "product":
        E, M, K = case["experts"], case["rows"], case["cols"]
        n = max(1, round(case["tokens"] * case["top_k"] * case["local"]))
        used = E * (1 - (1 - 1 / E) ** n) if E > 1 else 1
        b = used * (M * K + 4 * _groups(M) * _groups(K)) + n * (K + 4 * _groups(K))
        return {"bytes": b + n * M * _size(case["y"]), "flops": 2 * n * M * K}
    if case["op"] == "act":
        n, s = case["rows"] * case["inter"], _size(case["x"])
        if case["grad"]:
            return {"bytes": 5 * s * n, "flops": 12 * n}
        return {"bytes": n * (2 * s + 1) + 4 * case["rows"] * _groups(case["inter"]), "flops": 8 * n}
    T, k, H, kept = case["tokens"], case["top_k"], case["hidden"], _kept(case)
    if case["op"] == "sort":
        row = H * _size(case["to"]) + (4 * _groups(H) if case["to"] == "fp8" else 0)
        return {"bytes": T * H * _size(case["x"]) + kept * row + 8 * T * k + 4 * case["experts"],
                "flops": T * H}
    token, row = H * _size(case["y"]), H * _size(case["rows"])
    if case["grad"]:
        return {"bytes": T * token + 2 * kept * row + 12 * T * k, "flops": 3 * kept * H}
    return {"bytes": T * token * (2 if case["resid"] else 1) + kept * row + 8 * T * k,
            "flops": 2 * kept * H}


# ---- inputs -------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)

    def codes(*shape, std):
        x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
        return x.mul_(std).clamp_(-TOP, TOP).to(E4M3)

    def scales(*shape, mean):
        return (torch.rand(*shape, generator=g, device=DEV) + 0.5) * mean

    s = dict(case=case)
    if case["op"] == "product":
        E, M, K = case["experts"], case["rows"], case["cols"]
        # how many rows each expert got: experts are not equally popular
        rng = np.random.default_rng(seed)
        n = case["tokens"] * case["top_k"]
        live = max(1, round(n * case["local"]))
        popular = np.exp(0.3 * rng.standard_normal(E))
        counts = rng.multinomial(live, popular / popular.sum())
        s["most"] = int(counts.max())
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32,
                                    device=DEV)
        # blocks of 128 x 128 weights of 0.02, rows of activations around 1
        s["w"], s["ws"] = codes(E, M, K, std=112.0), scales(E, _groups(M), _groups(K),
                                                            mean=0.02 / 112)
        s["q"], s["qs"] = codes(n, K, std=160.0), scales(n, _groups(K), mean=1 / 160)
        s["y"] = torch.zeros(n, M, dtype=DT[case["y"]], device=DEV)
        if own:
            from ainfer_amd import moe
            s["weights"] = moe.Fp8Weights(s["w"], s["ws"])
        return s
    if case["op"] == "act":
        n, I, dt = case["rows"], case["inter"], DT[case["x"]]
        # gate and up side by side, as one product writes them
        gu = normal(n, 2 * I, std=1.5, dtype=dt)
        s["gate"], s["up"] = gu[:, :I], gu[:, I:]
        if case["grad"]:
            s["dact"], s["dgu"] = normal(n, I, dtype=dt), torch.empty_like(gu)
        else:
            s["q"] = torch.empty(n, I, dtype=E4M3, device=DEV)
            s["qs"] = torch.empty(n, _groups(I), dtype=torch.float32, device=DEV)
        return s
    T, E, k, H = (case[n] for n in ("tokens", "experts", "top_k", "hidden"))
    s["idx"] = _routed(T, E + case["elsewhere"], k, g)
    if case["op"] == "sort":
        s["x"] = normal(T, H, dtype=DT[case["x"]])
        # what a program keeps: the rows' buffers (rows of dropped pairs stay as they are)
        if case["to"] == "fp8":
            s["rows"] = torch.zeros(T * k, H, dtype=E4M3, device=DEV)
            s["scales"] = torch.zeros(T * k, _groups(H), dtype=torch.float32, device=DEV)
        else:
            s["rows"] = torch.zeros(T * k, H, dtype=DT[case["x"]], device=DEV)
            s["scales"] = None
        s["offsets"] = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        s["pos"] = torch.zeros(T, k, dtype=torch.int32, device=DEV)
        if own:
            from ainfer_amd import moe
            s["work"] = moe.sort_workspace(T, k, E)
        return s
    s["pos"] = _sorted(s["idx"], E)[2]
    s["rows"] = normal(T * k, H, dtype=DT[case["rows"]])
    w = torch.rand(T, k, generator=g, device=DEV) + 0.05
    s["w"] = w / w.sum(1, keepdim=True)
    if case["grad"]:
        s["dy"] = normal(T, H, dtype=DT[case["y"]])
        s["drows"] = torch.zeros_like(s["rows"])
        s["dw"] = torch.empty(T, k, dtype=torch.float32, device=DEV)
    else:
        s["resid"] = normal(T, H, dtype=DT[case["y"]]) if case["resid"] else None
        s["y"] = torch.empty(T, H, dtype=DT[case["y"]], device=DEV)
    return s


def _routed(T, E, k, g):
    """k distinct experts a token, some of them more popular."""
    popular = torch.randn(E, generator=g, device=DEV) * 0.5
    noise = torch.rand(T, E, generator=g, device=DEV).clamp_min_(1e-9)
    return (popular - torch.log(-torch.log(noise))).topk(k, 1)[1].to(torch.int32).contiguous()


# ---- one pass -------------------------------------------------------------------

def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from ainfer_amd import moe
        if op == "product":
            s["weights"].product(s["q"], s["qs"], s["y"], s["offsets"])
        elif op == "sort":
            moe.sort_rows(s["x"], s["idx"], case["experts"], s["work"], pow2=case["pow2"],
                          out=(s["rows"], s["scales"], s["offsets"], s["pos"]))
        elif op == "back" and case["grad"]:
            moe.unpermute_backward(s["dy"], s["rows"], s["pos"], s["w"], s["drows"], s["dw"])
        elif op == "back":
            moe.unpermute(s["rows"], s["pos"], s["w"], s["y"], resid=s["resid"])
        elif case["grad"]:
            I = case["inter"]
            moe.silu_mul_backward(s["dact"], s["gate"], s["up"], s["dgu"][:, :I], s["dgu"][:, I:])
        else:
            moe.silu_mul_fp8(s["gate"], s["up"], s["q"], s["qs"], pow2=case["pow2"])
    elif op == "product":
        _plain_product(s)
    elif op == "sort":
        _plain_sort(s)
    elif op == "back":
        _plain_back(s)
    else:
        _plain_act(s)
    return {"product": lambda: s["y"],
            "sort": lambda: [t for t in (s["rows"], s["scales"], s["offsets"], s["pos"])
                             if t is not None],
            "back": lambda: (s["drows"], s["dw"]) if case["grad"] else s["y"],
            "act": lambda: s["dgu"] if case["grad"] else (s["q"], s["qs"])}[op]()


def _wide(scales, dim, n):
    """Each scale for the values that it stands for: 128 along `dim`."""
    return scales.repeat_interleave(128, dim).narrow(dim, 0, n)


def _plain_product(s):
    case = s["case"]
    E, M, K = case["experts"], case["rows"], case["cols"]
    w = s["w"].float() * _wide(_wide(s["ws"], 2, K), 1, M)
    x = s["q"].float() * _wide(s["qs"], 1, K)
    if E == 1:
        n = s["most"]
        s["y"][:n] = (x[:n] @ w[0].t()).to(s["y"].dtype)
        return
    # the experts' rows side by side, as many places each as the busiest needs
    start, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    at = start[:, None] + torch.arange(s["most"], device=DEV)
    there = at < end[:, None]
    y = torch.bmm(x[at.clamp_max(x.shape[0] - 1)], w.transpose(1, 2).contiguous())
    # places behind an expert's last row go to a row that is left out
    to = torch.where(there, at, x.shape[0])
    wide = torch.cat([s["y"], s["y"][:1]])
    wide[to.flatten()] = y.flatten(0, 1).to(s["y"].dtype)
    s["y"].copy_(wide[:-1])


def _sorted(idx, E):
    """offsets [E + 1], order [T * k] (pair of each place, dropped ones last), pos [T][k]."""
    key = idx.flatten().long()
    key = torch.where((key >= 0) & (key < E), key, E)
    in_order, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(in_order, torch.arange(E + 1, device=DEV)).to(torch.int32)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=DEV)
    pos = torch.where(key < E, pos, -1).view(idx.shape).to(torch.int32)
    return offsets, order, pos


def _quantised(x, pow2):
    """e4m3 codes of fp32 rows and their scales, one for 128 columns."""
    n, K = x.shape
    blocks = torch.nn.functional.pad(x, (0, -K % 128)).view(n, -1, 128)
    most = blocks.abs().amax(2)
    scale = (most / TOP).clamp_min(LEAST)
    if pow2:  # the next power of two that is not below it
        fraction, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (fraction == 0.5).to(torch.int32))
    scale = torch.where(most == 0, 1.0, scale)
    q = (blocks / scale[:, :, None]).view(n, -1)[:, :K].to(E4M3)
    return q, scale


def _plain_sort(s):
    case = s["case"]
    E, k = case["experts"], case["top_k"]
    offsets, order, pos = _sorted(s["idx"], E)
    s["offsets"].copy_(offsets)
    s["pos"].copy_(pos)
    live = (torch.arange(order.numel(), device=DEV) < offsets[-1])[:, None]
    token = order // k
    if case["to"] == "fp8":
        q, scale = _quantised(s["x"].float(), case["pow2"])
        rows = s["rows"].view(torch.uint8)
        rows.copy_(torch.where(live, q.view(torch.uint8)[token], rows))
        s["scales"].copy_(torch.where(live, scale[token], s["scales"]))
    else:
        s["rows"].copy_(torch.where(live, s["x"][token], s["rows"]))


def _plain_back(s):
    pos = s["pos"].long()
    there = pos >= 0
    rows = s["rows"].float()
    mine = rows[pos.clamp_min(0)]
    w = torch.where(there, s["w"], 0.0)
    if not s["case"]["grad"]:
        y = torch.where(there[:, :, None], mine * w[:, :, None], 0.0).sum(1)
        if s["resid"] is not None:
            y = y + s["resid"].float()
        s["y"].copy_(y)
        return
    dy = s["dy"].float()
    s["dw"].copy_(torch.where(there, (mine * dy[:, None, :]).sum(2), 0.0))
    n = rows.shape[0]
    to = torch.where(there, pos, n).flatten()
    wide = torch.cat([s["drows"], s["drows"][:1]])
    wide[to] = (w[:, :, None] * dy[:, None, :]).flatten(0, 1).to(wide.dtype)
    s["drows"].copy_(wide[:-1])


def _plain_act(s):
    g, u = s["gate"].float(), s["up"].float()
    sig = 1 / (1 + torch.exp(-g))
    if s["case"]["grad"]:
        d = s["dact"].float()
        s["dgu"].copy_(torch.cat([d * u * sig * (1 + g * (1 - sig)), d * g * sig], 1))
        return
    q, scale = _quantised(g * sig * u, s["case"]["pow2"])
    s["q"].view(torch.uint8).copy_(q.view(torch.uint8))
    s["qs"].copy_(scale)


# ---- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"product": _exact_product, "sort": _exact_sort, "back": _exact_back,
            "act": _exact_act}[case["op"]](case, s)


def _exact_product(case, s):
    M, K = case["rows"], case["cols"]
    y = s["y"].double()
    of_row = torch.arange(M, device=DEV) // 128
    of_col = torch.arange(K, device=DEV) // 128
    bounds = s["offsets"].tolist()
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if b > a:
            w = s["w"][e].double() * s["ws"][e].double()[of_row][:, of_col]
            x = s["q"][a:b].double() * s["qs"][a:b].double()[:, of_col]
            y[a:b] = x @ w.t().contiguous()
    return y


def _exact_codes(x, pow2):
    """The definition's codes and scales of 64-bit rows, and the codes as values."""
    n, K = x.shape
    q, scales = torch.empty(n, K, dtype=torch.float64, device=DEV), []
    for c in range(0, K, 128):
        part = x[:, c:c + 128]
        most = part.abs().max(1).values
        scale = torch.clamp(most / TOP, min=LEAST)
        if pow2:
            scale = torch.exp2(torch.ceil(torch.log2(scale)))
        scale = torch.where(most > 0, scale, torch.ones_like(scale))
        v = part / scale[:, None]
        # the nearest multiple of the value's step, ties to even ones; 2^-9 is the least
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp_min(1e-30))), min=-6.0)
                          - 3)
        q[:, c:c + 128] = torch.clamp(torch.round(v / step) * step, -TOP, TOP)
        scales.append(scale)
    return q, torch.stack(scales, 1)


def _exact_sort(case, s):
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    ids = s["idx"].cpu().numpy().reshape(-1)
    pairs = [np.flatnonzero(ids == e) for e in range(E)]
    offsets = np.concatenate([[0], np.cumsum([len(p) for p in pairs])])
    at = np.concatenate(pairs)
    pos = np.full(T * k, -1)
    pos[at] = np.arange(len(at))
    token = torch.tensor(at // k, device=DEV)
    out = []
    if case["to"] == "fp8":
        for t, kept in zip(_exact_codes(s["x"].double(), case["pow2"]), (s["rows"], s["scales"])):
            kept = kept.double()
            kept[:len(at)] = t[token]
            out.append(kept)
    else:
        out.append(s["rows"].double())
        out[0][:len(at)] = s["x"].double()[token]
    return out + [torch.tensor(offsets, dtype=torch.int32),
                  torch.tensor(pos, dtype=torch.int32).view(T, k)]


def _exact_back(case, s):
    T, k = case["tokens"], case["top_k"]
    if case["grad"]:
        drows = s["drows"].double()
        dw = torch.zeros(T, k, dtype=torch.float64, device=DEV)
    else:
        y = torch.zeros(T, case["hidden"], dtype=torch.float64, device=DEV)
        if s["resid"] is not None:
            y += s["resid"].double()
    for j in range(k):
        t = torch.nonzero(s["pos"][:, j] >= 0)[:, 0]
        p, w = s["pos"][t, j].long(), s["w"][t, j].double()
        row = s["rows"][p].double()
        if case["grad"]:
            dy = s["dy"][t].double()
            drows[p] = w[:, None] * dy
            dw[t, j] = torch.linalg.vecdot(row, dy)
        else:
            y[t] += w[:, None] * row
    return (drows, dw) if case["grad"] else y


def _exact_act(case, s):
    g, u = s["gate"].double(), s["up"].double()
    if case["grad"]:
        d, y = s["dact"].double(), torch.nn.functional.silu(g)
        sig = torch.sigmoid(g)
        return torch.cat([d * u * (sig + y * (1 - sig)), d * y], 1)
    return _exact_codes(g * torch.sigmoid(g) * u, case["pow2"])
