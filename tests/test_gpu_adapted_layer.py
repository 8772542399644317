"""The operators around the expert stage run together, as a server would: a
layer's router logits scored in groups, its experts, the shared expert with each
token's adapters, combine.  Every stage is checked against its formula in 64
bits on the inputs it had in the run; the composed calls then have to give the
staged run's bits, on another stream and from a replayed graph too.

Tolerances: those of the single operators' tests; combine is a chain of k + 1
fp32 fma (2^-24 of the magnitudes each) and one rounding to bf16 (2^-8)."""
import dataclasses
from types import SimpleNamespace

import numpy as np
import pytest

import test_gpu_lora as TL
import test_gpu_scored as TS

pytestmark = pytest.mark.gpu

N = 5


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def world(torch):
    from ainfer_amd import _lib as L
    from ainfer_amd.moe import LoraAdapters, MoeLayer
    from ainfer_amd.synthetic import CONFIGS
    layer = MoeLayer(dataclasses.replace(CONFIGS["c0"], zipf=0.7))
    H, I, R = 1024, 256, 24
    g = torch.Generator(device="cuda")
    g.manual_seed(11)

    def normal(*s, std):
        return (torch.randn(*s, generator=g, device="cuda") * std).bfloat16()

    ranks = torch.tensor([24, 8, 0, 16, 13], dtype=torch.int32, device="cuda")
    scales = torch.rand(N, generator=g, device="cuda") + 0.5
    gu = LoraAdapters([normal(N, R, H, std=0.03) for _ in range(2)],
                      [normal(N, I, R, std=0.2) for _ in range(2)], ranks=ranks, scales=scales,
                      y_dtype=torch.float32)
    down = LoraAdapters([normal(N, R, I, std=0.06)], [normal(N, H, R, std=0.2)], ranks=ranks,
                        scales=scales, x_dtype=torch.float32, y_dtype=torch.float32)
    bias = torch.randn(64, generator=g, device="cuda") * 0.1
    r = L.Routing(64, 8, L.SCORE_SIGMOID, 8, 4, L.GROUP_TOP2, 1, 2.5)
    return SimpleNamespace(layer=layer, gu=gu, down=down, bias=bias, r=r, ranks=ranks,
                           scales=scales, R=R)


def inputs(torch, w, T, tag):
    from ainfer_amd.moe import make_input
    x = make_input(w.layer.cfg, T, tag=tag)
    ids = torch.tensor([(7 * t + tag) % (N + 1) - 1 for t in range(T)], dtype=torch.int32,
                       device="cuda")
    wsl = max((w.gu.workspace(T), w.down.workspace(T)), key=lambda t: t.numel())
    return x, ids, wsl, w.layer.workspace(min(T, 4096))


def together(w, x, ids, wsl, ws, y, resid=None, stream=None):
    shared = w.layer.shared_adapted(x, ids, w.gu, w.down, wsl, stream=stream)
    w.layer.forward_scored(x, y, ws, w.r, w.bias, resid=resid, shared=shared, stream=stream)
    return y


def check_lora(torch, w, lora, x, ids, before, after):
    a, b, _, _ = lora.tensors
    TL.Case.compare(SimpleNamespace(torch=torch, ids=ids, T=x.shape[0], N=N, R=w.R, K=x.shape[1],
                                    Ms=lora.rows, a=a, b=b, x=x, ranks=w.ranks,
                                    scales=w.scales), before, after)


@pytest.mark.parametrize("T", (1, 2, 7, 33, 300))
def test_stages_and_composition(torch, world, T):
    from ainfer_amd import moe
    w, layer, sh = world, world.layer, world.layer.shape
    print(f"[case] scored and adapted layer T={T}", flush=True)
    x, ids, wsl, ws = inputs(torch, w, T, T)
    resid = x.flip(0).contiguous()

    idx, wt, sg, logits = layer.route(x, ws, want_logits=True)
    idx, wt = moe.route_scored(w.r, logits, w.bias)
    torch.cuda.synchronize()
    ri, rw = TS.reference(logits.double().cpu().numpy(), torch.finfo(torch.float32).min,
                          w.bias.cpu().numpy(), 64, 8, w.r.score, 8, 4, w.r.group_score, 1, 2.5)
    assert np.array_equal(idx.cpu().numpy(), ri)
    assert np.all(np.abs(wt.cpu().numpy() - rw) <= TS.RTOL * np.abs(rw) + TS.ATOL)

    q, sq = moe.act_quant_i8(x)
    gate = moe.int4_gemv_i8(layer.weights.ws_gate, layer.weights.ss_gate, sh.scale_dtype, q, sq,
                            256)
    up = moe.int4_gemv_i8(layer.weights.ws_up, layer.weights.ss_up, sh.scale_dtype, q, sq, 256)
    before = [gate.clone(), up.clone()]
    w.gu.apply(x, ids, [gate, up], wsl)
    torch.cuda.synchronize()
    check_lora(torch, w, w.gu, x, ids, before, [gate, up])
    act = moe.silu_mul(gate, up, torch.empty_like(gate))
    want = gate.double() / (1 + (-gate.double()).exp()) * up.double()
    assert ((act.double() - want).abs() <= 2.0 ** -21 * want.abs() + 1e-37).all()
    q, sq = moe.act_quant_i8(act)
    out = moe.int4_gemv_i8(layer.weights.ws_down, layer.weights.ss_down, sh.scale_dtype, q, sq,
                           1024)
    before = [out.clone()]
    w.down.apply(act, ids, [out], wsl)
    torch.cuda.synchronize()
    check_lora(torch, w, w.down, act, ids, before, [out])

    o = layer.experts(x, idx, ws)
    o[T * 8:] = out.bfloat16()
    y = torch.empty_like(x)
    layer.combine(o, wt, sg, y, resid)
    torch.cuda.synchronize()
    od = o.double()
    terms = torch.cat([od[:T * 8].view(T, 8, 1024) * wt.double()[:, :, None],
                       (od[T * 8:] * sg.double()[:, None])[:, None],
                       resid.double()[:, None]], 1)
    want, mag = terms.sum(1), terms.abs().sum(1)
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 11 * 2.0 ** -24 * 1.01 * mag).all()

    got = together(w, x, ids, wsl, ws, torch.empty_like(x), resid)
    torch.cuda.synchronize()
    assert torch.equal(got.view(torch.int16), y.view(torch.int16))
    assert layer.workspace_check(ws) == 0


def test_without_adapters_and_without_shared_rows(torch, world):
    """No adapter on any token changes nothing; without shared rows the layer's
    own shared expert is combined."""
    w, T = world, 20
    print("[case] scored layer without adapters", flush=True)
    x, ids, wsl, ws = inputs(torch, w, T, 3)
    plain = w.layer.shared_adapted(x, ids, None, None, wsl)
    none = w.layer.shared_adapted(x, torch.full_like(ids, -1), w.gu, w.down, wsl)
    assert torch.equal(plain.view(torch.int16), none.view(torch.int16))
    y = w.layer.forward_scored(x, torch.empty_like(x), ws, w.r, w.bias)
    idx, _, sg, logits = w.layer.route(x, ws, want_logits=True)
    from ainfer_amd import moe
    idx, wt = moe.route_scored(w.r, logits, w.bias)
    want = w.layer.combine(w.layer.experts(x, idx, ws), wt, sg, torch.empty_like(x))
    assert torch.equal(y.view(torch.int16), want.view(torch.int16))


def test_more_tokens_than_a_chunk(torch, world):
    w, T = world, 4096 + 21
    print(f"[case] scored and adapted layer T={T}", flush=True)
    x, ids, wsl, ws = inputs(torch, w, T, 9)
    y = together(w, x, ids, wsl, ws, torch.empty_like(x))
    shared = w.layer.shared_adapted(x, ids, w.gu, w.down, wsl)
    for c in (slice(0, 4096), slice(4096, T)):
        part = w.layer.forward_scored(x[c], torch.empty_like(x[c]), ws, w.r, w.bias,
                                      shared=shared[c])
        assert torch.equal(part.view(torch.int16), y[c].view(torch.int16))


@pytest.mark.parametrize("T", (1, 24))
def test_other_stream_and_replayed_graph(torch, world, T):
    """Captured once and replayed on new inputs, with eager work between the
    replays, each replay against the eager run."""
    w = world
    print(f"[case] scored and adapted layer in a graph T={T}", flush=True)
    x, ids, wsl, ws = inputs(torch, w, T, 40)
    y = torch.empty_like(x)
    s = torch.cuda.Stream()
    want = together(w, x, ids, wsl, ws, torch.empty_like(x))
    s.wait_stream(torch.cuda.current_stream())
    together(w, x, ids, wsl, ws, y, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(y.view(torch.int16), want.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        together(w, x, ids, wsl, ws, y)
    for i in range(4):
        x2, ids2, _, _ = inputs(torch, w, T, 50 + i)
        x.copy_(x2)
        ids.copy_(ids2)
        y.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        want = together(w, x2, ids2, wsl, ws, torch.empty_like(x))
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), i


def test_refusals(torch, world):
    from ainfer_amd import _lib as L
    w, T = world, 3
    x, ids, wsl, ws = inputs(torch, w, T, 1)
    y = torch.empty_like(x)
    other = L.Routing(64, 4, w.r.score, 1, 1, 0, 1, 1.0)
    for call in (lambda: w.layer.forward_scored(x, y, ws, other),
                 lambda: w.layer.forward_scored(x, y[:2], ws, w.r),
                 lambda: w.layer.forward_scored(x.float(), y, ws, w.r),
                 lambda: w.layer.forward_scored(x, y, ws, w.r, shared=y.float()),
                 lambda: w.layer.forward_scored(x, y, ws, w.r, bias=w.bias[:63]),
                 lambda: w.layer.shared_adapted(x[:, :512], ids, None, None, wsl),
                 lambda: w.layer.shared_adapted(x, ids[:2], w.gu, None, wsl),
                 lambda: w.layer.shared_adapted(x, ids, w.down, None, wsl),
                 lambda: w.layer.shared_adapted(x, ids, w.gu, None, wsl[:16])):
        with pytest.raises(L.MoeError):
            call()


def test_no_tokens(torch, world):
    w = world
    x, ids, wsl, ws = inputs(torch, w, 1, 1)
    empty = torch.empty(0, 1024, dtype=torch.bfloat16, device="cuda")
    rows = w.layer.shared_adapted(empty, ids[:0], w.gu, w.down, wsl)
    assert rows.shape == (0, 1024)
    y = w.layer.forward_scored(empty, torch.empty_like(empty), ws, w.r, w.bias, shared=rows)
    assert y.shape == (0, 1024)
