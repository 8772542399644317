"""Scored routing (ainfer_moe_route_scored) against its definition in 64 bits.

Bar: expert indices equal; weights within RTOL of the 64-bit value.  The weights
are a few fp32 operations: the hardware's exp2 of an argument off by 1.125 2^-23 of
itself in all ((1.125 d + 1) 2^-23 for exp(-d), d up to 80: 2^-16.5; larger ones are
covered by ATOL), reciprocals to 2^-22, sums of at most 1024 positive terms, which
carry the errors of their large ones (2^-19): below 2^-16 in all.
ATOL covers what fp32 cannot hold (values below its normal range)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
RTOL, ATOL = 2.0 ** -16, 1e-36

SOFT, SIG = 0, 1
GMAX, GTOP2 = 0, 1


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def reference(logits, lowest, bias, E, k, score, G, top, gscore, renorm, scale):
    """One token at a time, as the header defines it, in 64 bits."""
    out_i, out_w = [], []
    for row in logits:
        l = np.asarray(row, dtype=np.float64)
        masked = ~(l > lowest)                      # NaN too
        b = np.zeros(E) if bias is None else np.asarray(bias, dtype=np.float64)
        if bias is not None:
            masked = masked | np.isnan(b) | (b == -np.inf)
            b = np.where(masked, 0.0, np.clip(b, -float(np.float32(1e38)), float(np.float32(1e38))))
        l = np.where(masked, 0.0, np.minimum(l, float(np.finfo(np.float32).max)))
        lm = np.where(~(np.asarray(row, dtype=np.float64) > lowest), -np.inf,
                      np.minimum(np.asarray(row, dtype=np.float64), float(np.finfo(np.float32).max)))
        with np.errstate(over="ignore"):
            if score == SIG:
                s = 1 / (1 + np.exp(-l))
            else:
                m = lm.max() if np.isfinite(lm.max()) else 0.0
                e = np.where(np.isfinite(lm), np.exp(np.where(np.isfinite(lm), lm - m, -np.inf)), 0)
                s = e / e.sum() if e.sum() > 0 else np.zeros(E)
        key = np.where(masked, -np.inf, l if bias is None else s + b)
        both = np.where(masked, -np.inf, s + b)
        groups = []
        for g in range(G):
            own = slice(g * (E // G), (g + 1) * (E // G))
            if gscore == GMAX:
                groups.append(key[own].max())
            else:
                two = sorted(both[own])[::-1][:2]
                two = [v for v in two if v > -np.inf]
                groups.append(sum(two) if two else -np.inf)
        kept = sorted(range(G), key=lambda g: (-groups[g], g))[:top] if G > 1 else [0]
        mine = [e for e in range(E) if e // (E // G) in kept]
        pick = sorted(mine, key=lambda e: (-key[e], e))[:k]
        w = np.array([0.0 if masked[e] else s[e] for e in pick])
        if renorm:
            # logits far below zero leave no normal score: their ratios are exp's
            lp = np.array([l[e] for e in pick])
            live = np.array([not masked[e] for e in pick])
            if live.any():
                if score == SIG:
                    logs = np.where(lp > 0, -np.log1p(np.exp(-np.abs(lp))),
                                    lp - np.log1p(np.exp(-np.abs(lp))))
                else:
                    logs = lp
                w = np.where(live, np.exp(np.where(live, logs - logs[live].max(), -np.inf)), 0.0)
                w = w / w.sum()
            else:
                w = np.zeros(len(pick))
        out_i.append(pick)
        out_w.append(w * scale)
    return np.array(out_i), np.array(out_w)


def run(torch, logits, bias, k, score, G=1, top=1, gscore=GTOP2, renorm=1, scale=1.0, stream=None):
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    r = L.Routing(logits.shape[1], k, score, G, top, gscore, renorm, scale)
    idx, w = moe.route_scored(r, logits, bias, stream=stream)
    torch.cuda.synchronize()
    return idx.cpu().numpy(), w.cpu().numpy()


def check(torch, logits, bias, k, score, G=1, top=1, gscore=GTOP2, renorm=1, scale=1.0):
    T, E = logits.shape
    print(f"[case] T={T} E={E} k={k} score={score} G={G}/{top} gs={gscore} renorm={renorm} "
          f"{logits.dtype} bias={bias is not None} ld={logits.stride(0)}", flush=True)
    idx, w = run(torch, logits, bias, k, score, G, top, gscore, renorm, scale)
    lowest = torch.finfo(logits.dtype).min
    ri, rw = reference(logits.double().cpu().numpy(), lowest,
                       None if bias is None else bias.cpu().numpy(), E, k, score, G, top, gscore,
                       renorm, scale)
    assert np.array_equal(idx, ri)
    assert np.all(np.abs(w - rw) <= RTOL * np.abs(rw) + ATOL * max(1.0, abs(scale)))


def logits_of(torch, T, E, dtype, seed, std=1.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(T, E, generator=g, device="cuda") * std).to(dtype)


# (T, E, k, groups, kept): one token to a few hundred, one expert to 1024, groups of
# one to 512 experts in every lane layout, one to 64 groups
SHAPES = [(1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (7, 60, 4, 6, 3), (333, 64, 8, 1, 1),
          (130, 512, 10, 1, 1), (65, 1024, 32, 1, 1), (33, 1024, 32, 64, 8), (5, 23, 13, 1, 1),
          (40, 96, 6, 3, 2), (9, 1023, 7, 33, 5), (17, 960, 16, 48, 3), (64, 40, 1, 8, 1),
          (12, 64, 6, 64, 6), (30, 873, 9, 3, 1), (30, 864, 9, 3, 2), (19, 300, 11, 1, 1), (21, 1024, 9, 2, 1), (3, 65, 32, 5, 3), (257, 160, 8, 8, 3)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("score", (SOFT, SIG))
@pytest.mark.parametrize("biased", (False, True))
def test_matches_definition(torch, shape, score, biased):
    T, E, k, G, top = shape
    seed = T * 1000 + E + score
    for dtype, gscore, renorm in ((torch.float32, GTOP2, 1), (torch.bfloat16, GMAX, 0),
                                  (torch.float32, GMAX, 0), (torch.bfloat16, GTOP2, 1)):
        x = logits_of(torch, T, E, dtype, seed)
        bias = None
        if biased:
            bias = logits_of(torch, 1, E, torch.float32, seed + 7, 0.1 if score == SIG else 1 / E)[0]
        check(torch, x, bias, k, score, G, top, gscore, renorm, 2.5)


@pytest.mark.parametrize("score", (SOFT, SIG))
@pytest.mark.parametrize("biased", (False, True))
@pytest.mark.parametrize("G,top", ((1, 1), (4, 2), (16, 3)))
def test_masks_infinities_and_ties(torch, score, biased, G, top):
    """Rows whose mask leaves nothing, one or a few experts; the type's lowest
    value, infinities and NaN; equal logits (more than 64 of them); signed zeros."""
    E, k = 256, 8
    for dtype in (torch.float32, torch.bfloat16):
        lowest = torch.finfo(dtype).min
        x = logits_of(torch, 16, E, dtype, 5)
        x[0] = -math.inf
        x[1] = lowest
        x[2] = math.nan
        x[3] = -math.inf
        x[3, 100] = 0.5
        x[4, :250] = lowest
        x[5] = 0.0
        x[6, ::2] = 0.0
        x[6, 1::2] = -0.0
        x[7, [3, 9, 200]] = math.inf
        x[8, ::3] = math.nan
        x[8, 1::3] = -math.inf
        x[9] = -90.0
        x[9, 20:40] = -88.5
        x[10] = 60.0
        x[11, 128:] = -math.inf
        x[12] = (x[12].float() * 8).round().to(dtype) / 8
        x[13] = x[13] * 1e4
        x[14] = -math.inf
        x[14, 64:68] = 1.0
        bias = None
        if biased:
            bias = logits_of(torch, 1, E, torch.float32, 3, 0.05)[0]
            bias[[5, 70]] = -math.inf
            bias[9] = math.nan
            bias[[130, 250]] = math.inf
        for gscore in (GMAX, GTOP2):
            for renorm in (0, 1):
                check(torch, x, bias, k, score, G, top, gscore, renorm, 1.0)


@pytest.mark.parametrize("score", (SOFT, SIG))
@pytest.mark.parametrize("near", (12, 40, 512))
def test_keys_nearer_than_fp32(torch, score, near):
    """Biases that bring `near` experts' keys within an fp32 step of one value: the
    order is that of the 64-bit keys."""
    E, k = 512, 10
    x = logits_of(torch, 1, E, torch.float32, near)
    d = x[0].double()
    s = torch.sigmoid(d) if score == SIG else torch.softmax(d, 0)
    bias = torch.full((E,), -2.0, device="cuda")
    at = torch.randperm(E, generator=torch.Generator().manual_seed(near))[:near].cuda()
    bias[at] = (0.75 - s[at]).float()
    check(torch, x, bias, k, score)
    check(torch, x, bias, k, score, 8, 3, GTOP2)
    check(torch, x, bias, k, score, 8, 3, GMAX)


def test_group_values_nearer_than_fp32(torch):
    """Groups whose two largest keys sum to one value but for the last bits."""
    E, G = 128, 8
    x = logits_of(torch, 6, E, torch.float32, 77)
    s = torch.sigmoid(x.double())
    for t in range(6):
        bias = torch.full((E,), -1.0, device="cuda")
        for g in range(G):
            own = torch.arange(g * 16, g * 16 + 2, device="cuda")
            bias[own] = (0.5 - s[t, own]).float()
        check(torch, x[t:t + 1], bias, 4, SIG, G, 3, GTOP2)
        check(torch, x[t:t + 1], bias, 4, SIG, G, 3, GMAX)


def test_row_pitch_and_alignment(torch):
    wide = logits_of(torch, 37, 300, torch.float32, 1)
    for off, n in ((0, 256), (1, 256), (3, 60), (4, 128)):
        check(torch, wide[:, off:off + n], None, 4, SIG, 4, 2)
    half = logits_of(torch, 37, 304, torch.bfloat16, 2)
    for off, n in ((0, 256), (1, 256), (8, 128), (2, 60)):
        check(torch, half[:, off:off + n], None, 4, SOFT, 4, 2)
    one = logits_of(torch, 1, 256, torch.float32, 3)
    check(torch, one, None, 8, SIG)


def test_large_call_and_offsets(torch):
    """65536 tokens on a pitch that passes 32 bits of elements; rows outside
    the tokens stay as they were."""
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    T, E, k, pitch = 65536, 16, 3, 70000
    store = torch.empty((T - 1) * pitch + E, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((T, E), (pitch, 1))
    x.copy_(logits_of(torch, T, E, torch.bfloat16, 4))
    idx, w = moe.route_scored(L.Routing(E, k, SIG, 1, 1, 0, 1, 1.0), x)
    dense = x.contiguous()
    del store, x
    idx2, w2 = moe.route_scored(L.Routing(E, k, SIG, 1, 1, 0, 1, 1.0), dense)
    assert torch.equal(idx, idx2) and torch.equal(w, w2)
    key = dense.double()
    ri = key.sort(dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(idx.long(), ri)
    big = torch.full((9, k), -5, dtype=torch.int32, device="cuda")
    wb = torch.full((9, k), -5.0, device="cuda")
    moe.route_scored(L.Routing(E, k, SIG, 1, 1, 0, 1, 1.0), dense[:6], out=(big[:6], wb[:6]))
    assert (big[6:] == -5).all() and (wb[6:] == -5).all() and torch.equal(big[:6], idx[:6])
    e = moe.route_scored(L.Routing(E, k, SIG, 1, 1, 0, 1, 1.0), dense[:0])
    assert e[0].shape == (0, k)


def test_streams_and_graph(torch):
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    r = L.Routing(256, 8, SIG, 8, 4, GTOP2, 1, 2.5)
    x = logits_of(torch, 100, 256, torch.float32, 8)
    bias = logits_of(torch, 1, 256, torch.float32, 9, 0.1)[0]
    want = moe.route_scored(r, x, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = moe.route_scored(r, x, bias, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = (torch.empty_like(want[0]), torch.empty_like(want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.route_scored(r, x, bias, out=out)
    for rep in range(3):
        x.copy_(logits_of(torch, 100, 256, torch.float32, 20 + rep))
        out[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = moe.route_scored(r, x, bias)
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def check_many(torch, x, bias, k, score, G=1, top=1, gscore=GTOP2, renorm=1, scale=1.0,
               T=16400):
    """The rows of x over and over in a random order (many tokens of few experts
    share a wave): each the definition's answer, whatever stands beside it."""
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    B, E = x.shape
    print(f"[case] T={T} of {B} rows E={E} k={k} score={score} G={G}/{top} gs={gscore} "
          f"renorm={renorm} {x.dtype} bias={bias is not None}", flush=True)
    order = torch.randint(0, B, (T,), generator=torch.Generator().manual_seed(B + E + k))
    order[-B:] = torch.arange(B)
    wide = torch.empty(T, E + 3, dtype=x.dtype, device="cuda")
    idx, w = [], []
    for rows in (x[order.cuda()], wide[:, 1:E + 1].copy_(x[order.cuda()])):
        out = (torch.full((T + 2, k), -7, dtype=torch.int32, device="cuda"),
               torch.full((T + 2, k), -7.0, device="cuda"))
        moe.route_scored(L.Routing(E, k, score, G, top, gscore, renorm, scale), rows, bias,
                         out=(out[0][:T], out[1][:T]))
        torch.cuda.synchronize()
        assert (out[0][T:] == -7).all() and (out[1][T:] == -7).all()
        idx.append(out[0][:T].cpu().numpy())
        w.append(out[1][:T].cpu().numpy())
    ri, rw = reference(x.double().cpu().numpy(), torch.finfo(x.dtype).min,
                       None if bias is None else bias.cpu().numpy(), E, k, score, G, top, gscore,
                       renorm, scale)
    order = order.numpy()
    for i, v in zip(idx, w):
        assert np.array_equal(i, ri[order])
        assert np.all(np.abs(v - rw[order]) <= RTOL * np.abs(rw[order]) + ATOL * max(1.0, abs(scale)))


@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (16, 3, 1, 1), (23, 13, 1, 1), (60, 4, 6, 3),
                                   (64, 8, 1, 1), (40, 6, 8, 7), (128, 16, 1, 1), (96, 6, 3, 2),
                                   (128, 8, 8, 4), (120, 16, 5, 2), (64, 6, 16, 5), (127, 9, 1, 1),
                                   (32, 2, 2, 1), (128, 12, 16, 16)])
@pytest.mark.parametrize("score", (SOFT, SIG))
@pytest.mark.parametrize("biased", (False, True))
def test_many_tokens_of_few_experts(torch, shape, score, biased):
    E, k, G, top = shape
    for dtype, gscore, renorm, T in ((torch.float32, GTOP2, 1, 16400), (torch.bfloat16, GMAX, 0, 16387),
                                     (torch.float32, GMAX, 0, 65536), (torch.bfloat16, GTOP2, 1, 20001)):
        x = logits_of(torch, 50, E, dtype, E + k + score)
        bias = None
        if biased:
            bias = logits_of(torch, 1, E, torch.float32, E + 7, 0.1 if score == SIG else 1 / E)[0]
        check_many(torch, x, bias, k, score, G, top, gscore, renorm, 2.5, T)


@pytest.mark.parametrize("score", (SOFT, SIG))
@pytest.mark.parametrize("biased", (False, True))
@pytest.mark.parametrize("G,top", ((1, 1), (4, 2), (16, 3)))
def test_many_tokens_masks_infinities_and_ties(torch, score, biased, G, top):
    E, k = 128, 8
    for dtype in (torch.float32, torch.bfloat16):
        x = logits_of(torch, 16, E, dtype, 5)
        x[0] = -math.inf
        x[1] = torch.finfo(dtype).min
        x[2] = math.nan
        x[3] = -math.inf
        x[3, 100] = 0.5
        x[4, :122] = torch.finfo(dtype).min
        x[5] = 0.0
        x[6, ::2] = 0.0
        x[6, 1::2] = -0.0
        x[7, [3, 9, 120]] = math.inf
        x[8, ::3] = math.nan
        x[8, 1::3] = -math.inf
        x[9] = -90.0
        x[9, 20:40] = -88.5
        x[10] = 60.0
        x[11, 64:] = -math.inf
        x[12] = (x[12].float() * 8).round().to(dtype) / 8
        x[13] = x[13] * 1e4
        x[14] = -math.inf
        x[14, 62:66] = 1.0
        bias = None
        if biased:
            bias = logits_of(torch, 1, E, torch.float32, 3, 0.05)[0]
            bias[[5, 70]] = -math.inf
            bias[9] = math.nan
            bias[[30, 125]] = math.inf
        for gscore in (GMAX, GTOP2):
            for renorm in (0, 1):
                check_many(torch, x, bias, k, score, G, top, gscore, renorm)


@pytest.mark.parametrize("score", (SOFT, SIG))
@pytest.mark.parametrize("near", (3, 12, 40, 128))
def test_many_tokens_keys_nearer_than_fp32(torch, score, near):
    """One row whose biased keys lie within an fp32 step of one value, among others."""
    E, k = 128, 6
    x = logits_of(torch, 9, E, torch.float32, near)
    d = x[4].double()
    s = torch.sigmoid(d) if score == SIG else torch.softmax(d, 0)
    bias = torch.full((E,), -2.0, device="cuda")
    at = torch.randperm(E, generator=torch.Generator().manual_seed(near))[:near].cuda()
    bias[at] = (0.75 - s[at]).float()
    check_many(torch, x, bias, k, score)
    check_many(torch, x, bias, k, score, 8, 3, GTOP2)
    check_many(torch, x, bias, k, score, 8, 3, GMAX)


def test_many_tokens_group_values_nearer_than_fp32(torch):
    E, G = 128, 8
    x = logits_of(torch, 6, E, torch.float32, 77)
    s = torch.sigmoid(x.double())
    for t in range(6):
        bias = torch.full((E,), -1.0, device="cuda")
        for g in range(G):
            own = torch.arange(g * 16, g * 16 + 2, device="cuda")
            bias[own] = (0.5 - s[t, own]).float()
        check_many(torch, x, bias, 4, SIG, G, 3, GTOP2)
        check_many(torch, x, bias, 4, SIG, G, 3, GMAX)


def test_many_tokens_on_another_stream_and_in_a_graph(torch):
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    r = L.Routing(64, 6, SIG, 4, 2, GTOP2, 1, 2.5)
    x = logits_of(torch, 20000, 64, torch.float32, 8)
    bias = logits_of(torch, 1, 64, torch.float32, 9, 0.1)[0]
    want = moe.route_scored(r, x, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = moe.route_scored(r, x, bias, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    parts = [moe.route_scored(r, x[i:i + 999], bias) for i in range(0, 20000, 999)]
    assert torch.equal(torch.cat([p[0] for p in parts]), want[0])  # a wave a token: the same picks
    out = (torch.empty_like(want[0]), torch.empty_like(want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.route_scored(r, x, bias, out=out)
    for rep in range(3):
        x.copy_(logits_of(torch, 20000, 64, torch.float32, 20 + rep))
        out[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = moe.route_scored(r, x, bias)
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
