"""The shared expert's rows of shared_adapted (int8 activations) beside the layer's own
(bf16 activations, W4A16), and which tokens of a batch get which."""
import numpy as np
import pytest

from test_gpu_adapted_layer import inputs, torch, world  # noqa: F401  (the fixtures)

pytestmark = pytest.mark.gpu


def same(a, b, torch):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("T", (1, 5, 300))
def test_rows_without_adapters_beside_the_layers_own(torch, world, oracle, T):
    """Both are MLPs of the same INT4 weights.  In 64 bits g = Wg x, u = Wu x, act =
    g / (1 + exp(-g)) u, out = Wd act.  int8 codes of a group are off by half a step, s / 2,
    s the group's largest value / 127 (and 2^-21 of the value by the fp32 quotient); the
    gate's derivative is at most 1.1.  bf16: 2^-8.  fp32 sums of n terms: (n + 32) 2^-23 of
    the magnitudes, where a weight q enters at most as q + 136 in steps of its scale."""
    w, layer = world, world.layer
    H, I, k = 1024, 256, 8
    print(f"[case] shared rows T={T}", flush=True)
    x, ids, wsl, ws = inputs(torch, w, T, 60 + T)
    got = w.layer.shared_adapted(x, ids, None, None, wsl)
    idx = torch.arange(k, dtype=torch.int32, device="cuda").repeat(T, 1)
    own = layer.experts(x, idx, ws)[T * k:]
    torch.cuda.synchronize()

    def weight(name, rows, K):
        s = layer.t["ss_" + name].view(torch.int16).cpu().numpy().view(np.uint16)
        d = oracle.dequant(layer.t["ws_" + name].cpu().numpy(), s, layer.shape.scale_dtype, rows, K)
        scale = layer.t["ss_" + name].double().view(rows, K // 128).repeat_interleave(128, 1)
        return torch.from_numpy(np.asarray(d, np.float64)).cuda().view(rows, K), scale * 144

    def step(v):  # of a row's int8 groups, for each value; halved, and the quotient's rounding
        s = v.view(T, -1, 128).amax(2).repeat_interleave(128, 1) / 127
        return 0.5 * s * (1 + 2.0 ** -20) + 2.0 ** -21 * v

    def through(v, m):
        return v @ m.t().contiguous()

    (wg, og), (wu, ou), (wd, od) = weight("gate", I, H), weight("up", I, H), weight("down", H, I)
    xd = x.double()
    g, u = through(xd, wg), through(xd, wu)
    silu = g / (1 + (-g).exp())
    act = silu * u
    out = through(act, wd)
    eps = (H + 32) * 2.0 ** -23
    rows = []  # the two rows' distances from 64 bits
    for int8 in (True, False):
        dx = step(xd.abs()) if int8 else torch.zeros_like(xd)
        eg = through(dx, wg.abs()) + eps * through(xd.abs() + dx, og)
        eu = through(dx, wu.abs()) + eps * through(xd.abs() + dx, ou)
        ea = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu
        ea = ea + (2.0 ** -20 if int8 else 2.0 ** -8) * (act.abs() + ea)
        if int8:
            ea = ea + step(act.abs() + ea)
        eo = through(ea, wd.abs()) + eps * through(act.abs() + ea, od)
        rows.append(eo + 2.0 ** -8 * (out.abs() + eo))
    assert ((got.double() - out).abs() <= rows[0]).all()
    assert ((own.double() - out).abs() <= rows[1]).all()
    assert ((got.double() - own.double()).abs() <= rows[0] + rows[1]).all()
    rel = ((got.double() - own.double()).norm() / own.double().norm()).item()
    print(f"[case] relative distance {rel:.4f}", flush=True)
    assert not same(got, own, torch)  # and they do differ


@pytest.mark.parametrize("T", (1, 24, 4096 + 21))
def test_tokens_without_an_adapter_keep_the_layers_own_rows(torch, world, T):
    """shared_tokens: a token's result does not depend on who else has an adapter."""
    w = world
    print(f"[case] shared rows of some tokens T={T}", flush=True)
    x, ids, wsl, ws = inputs(torch, w, T, 70)
    shared = w.layer.shared_adapted(x, ids, w.gu, w.down, wsl)

    def run(**kw):
        return w.layer.forward_scored(x, torch.empty_like(x), ws, w.r, w.bias, resid=x, **kw)

    plain, every = run(), run(shared=shared)
    has = ids >= 0
    for mask in (has, torch.zeros_like(has), torch.ones_like(has)):
        y = run(shared=shared, shared_tokens=mask)
        assert same(y[mask], every[mask], torch) and same(y[~mask], plain[~mask], torch)


def test_in_a_graph_and_on_a_stream(torch, world):
    w, T = world, 24
    x, ids, wsl, ws = inputs(torch, w, T, 80)
    y, mask = torch.empty_like(x), torch.empty(T, dtype=torch.bool, device="cuda")

    def run(x, ids, mask, y, stream=None):
        torch.ge(ids, 0, out=mask)
        rows = w.layer.shared_adapted(x, ids, w.gu, w.down, wsl, stream=stream)
        return w.layer.forward_scored(x, y, ws, w.r, w.bias, shared=rows, shared_tokens=mask,
                                      stream=stream)

    want = run(x, ids, mask, torch.empty_like(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    run(x, ids, mask, y, stream=side)
    torch.cuda.synchronize()
    assert same(y, want, torch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(x, ids, mask, y)
    for i in range(3):
        x2, ids2, _, _ = inputs(torch, w, T, 81 + i)
        x.copy_(x2)
        ids.copy_(ids2)
        y.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        want = run(x2, ids2, torch.empty_like(mask), torch.empty_like(x))
        assert same(got, want, torch), i


def test_refusals(torch, world):
    from ainfer_amd import _lib as L
    w, T = world, 3
    x, ids, wsl, ws = inputs(torch, w, T, 1)
    y, mask = torch.empty_like(x), ids >= 0
    for kw in (dict(shared_tokens=mask), dict(shared=x, shared_tokens=mask[:2]),
               dict(shared=x, shared_tokens=ids), dict(shared=x, shared_tokens=mask.cpu()),
               dict(shared=x, shared_tokens=mask[:, None])):
        with pytest.raises(L.MoeError):
            w.layer.forward_scored(x, y, ws, w.r, **kw)
