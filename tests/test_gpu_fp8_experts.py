"""The 8-bit floating point experts composed: routed, sorted, two products with the
gated activation between, weighted and summed, and the gradients through all of it.

Bounds.  The chain gives the bits of its calls made one by one (each tested by itself).
Against 64 bits without the activations' codes: each code is off by 2^-4 of its value at
most, so an output that adds many of them is off by less than 2^-4 of its norm for each of
the two roundings it goes through, times 1.1, the gated activation's largest slope:
2 * 1.1 * 2^-4 = 0.14."""
import pytest

import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def experts(torch, E, H, I, pow2=False, y_dtype=None):
    """(experts with their transposed weights, the weights' 64-bit values)"""
    from ainfer_amd import moe
    g = torch.Generator(device="cuda")
    g.manual_seed(E + H)
    fwd, back, dense = [], [], []
    for M, K in ((2 * I, H), (H, I)):
        w = torch.randn(E, M, K, generator=g, device="cuda") * K ** -0.5
        q, s = moe.weight_quant_fp8(w, pow2)
        dt = y_dtype or torch.bfloat16
        fwd.append(moe.Fp8Weights(q, s, dt))
        back.append(moe.Fp8Weights(q, s, dt, transpose=True))
        dense.append(q.double() * R.wide(R.wide(s.double(), 2, K), 1, M))
    return moe.Fp8Experts(*fwd, back=back, pow2=pow2), dense


def routed(torch, T, k, E, H, dtype, seed=0):
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").to(dtype)
    logits = torch.randn(T, E, generator=g, device="cuda")
    idx, w = moe.route_scored(L.Routing(E, k, L.SCORE_SIGMOID, 1, 1, L.GROUP_MAX, 1, 1.5), logits)
    return x, idx, w


def plain(torch, ex, dense, x, idx, w):
    gu, dn = dense
    I = ex.inter
    y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for e in range(ex.n_experts):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if len(t):
            h = x[t].double() @ gu[e].t().contiguous()
            a = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
            y = y.index_add(0, t, w[t, j].double()[:, None] * (a @ dn[e].t().contiguous()))
    return y


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("T,k,E,H,I", ((1, 8, 16, 512, 256), (16, 4, 32, 272, 144), (300, 3, 8, 512, 128),
                                       (1000, 2, 4, 256, 400)))
def test_forward(torch, T, k, E, H, I, dtype):
    from ainfer_amd import moe
    print(f"[case] experts {T} {k} {E} {H} {I} {dtype}", flush=True)
    dt = getattr(torch, dtype)
    for pow2 in (False, True):
        ex, dense = experts(torch, E, H, I, pow2)
        x, idx, w = routed(torch, T, k, E, H, dt)
        idx[::3, 0] = E + 2  # experts of another GPU
        y = ex.forward(x, idx, w)
        ref = plain(torch, ex, dense, x, idx, w)
        assert (y.double() - ref).norm() <= 0.14 * ref.norm()
        q, sq, off, pos = moe.sort_rows(x, idx, E, moe.sort_workspace(T, k, E), fp8=True, pow2=pow2)
        h = ex.gate_up.product(q, sq, offsets=off)
        a, sa = moe.silu_mul_fp8(h[:, :I], h[:, I:], pow2=pow2, live=off)
        o = ex.down.product(a, sa, offsets=off)
        assert torch.equal(moe.unpermute(o, pos, w, torch.empty_like(x)), y)
        z = ex.forward(x, idx, w, y=x.clone(), resid=x)
        assert ((z.double() - x.double() - y.double()).abs()
                <= 2.0 ** -7 * (x.double().abs() + y.double().abs()) + 1e-6).all()


def test_no_tokens_and_no_kept_pairs(torch):
    ex, _ = experts(torch, 4, 256, 128)
    x, idx, w = routed(torch, 5, 2, 4, 256, torch.bfloat16)
    assert ex.forward(x[:0], idx[:0], w[:0]).shape == (0, 256)
    y, kept = ex.forward(x, torch.full_like(idx, 9), w, keep=True)
    assert (y == 0).all()
    dx, dw = ex.backward(torch.ones_like(x), kept)
    assert (dx == 0).all() and (dw == 0).all()
    z = ex.forward(x, torch.full_like(idx, -1), w, resid=x)
    assert torch.equal(z, x)


@pytest.mark.parametrize("T,k,E,H,I", ((1, 4, 8, 256, 128), (40, 4, 16, 272, 144), (500, 2, 4, 512, 256)))
def test_backward(torch, T, k, E, H, I):
    """dw against <dy, the rows that forward kept>, dx against the 64-bit chain from the
    kept rows, with the weights' values."""
    ex, (gu, dn) = experts(torch, E, H, I, y_dtype=torch.float32)
    x, idx, w = routed(torch, T, k, E, H, torch.float32)
    idx[::3, 0] = -1
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    dy = torch.randn(T, H, generator=g, device="cuda")
    y, kept = ex.forward(x, idx, w, keep=True)
    dx, dw = ex.backward(dy, kept)
    h, o, off, pos, _ = kept
    there = pos >= 0
    at = pos.clamp_min(0).long()
    terms = dy.double()[:, None, :] * o.double()[at]
    want = torch.where(there, terms.sum(2), 0.0)
    assert ((dw.double() - want).abs() <= (H + 8) * 2.0 ** -24 * terms.abs().sum(2) + 1e-30).all()
    ref = torch.zeros_like(dx, dtype=torch.float64)
    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if len(t):
            he = h.double()[pos[t, j].long()].requires_grad_()
            a = torch.nn.functional.silu(he[:, :I]) * he[:, I:]
            a.backward((w[t, j].double()[:, None] * dy[t].double()) @ dn[e])
            ref.index_add_(0, t, he.grad @ gu[e])
    assert (dx.double() - ref).norm() <= 0.14 * ref.norm()


def test_gradient_of_the_routing_weights_by_differences(torch):
    """The output is linear in w: one step is the slope."""
    ex, _ = experts(torch, 8, 256, 128, y_dtype=torch.float32)
    x, idx, w = routed(torch, 60, 3, 8, 256, torch.float32)
    dy = torch.randn(60, 256, device="cuda")
    y, kept = ex.forward(x, idx, w, keep=True)
    dw = ex.backward(dy, kept)[1]
    step = torch.randn_like(w)
    rise = (dy.double() * (ex.forward(x, idx, w + step).double() - y.double())).sum()
    slope = (dw.double() * step.double()).sum()
    assert abs(rise - slope) <= 1e-4 * (dw.double() * step.double()).abs().sum()


def test_captured_step(torch):
    """A forward and backward step in a graph, replayed on new tokens."""
    ex, _ = experts(torch, 8, 256, 128)
    for T in (2, 300):
        x, idx, w = routed(torch, T, 3, 8, 256, torch.bfloat16)
        dy = torch.randn(T, 256, device="cuda").to(torch.bfloat16)

        def step():
            y, kept = ex.forward(x, idx, w, keep=True)
            return (y, *ex.backward(dy, kept))

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for i in range(4):
            nx, ni, nw = routed(torch, T, 3, 8, 256, torch.bfloat16, seed=10 + i)
            x.copy_(nx), idx.copy_(ni), w.copy_(nw)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_over_its_input(torch):
    """y and resid may be x itself: the rows are sorted before anything is written."""
    ex, _ = experts(torch, 8, 256, 128)
    for T in (1, 7, 900):
        x, idx, w = routed(torch, T, 3, 8, 256, torch.bfloat16)
        want = ex.forward(x, idx, w, resid=x)
        z = x.clone()
        assert ex.forward(z, idx, w, y=z, resid=z) is z
        assert torch.equal(z, want)


def test_two_calls_at_once(torch):
    """Calls on two streams, of sizes that take each form of the sort and of the products, do not
    meet in anything."""
    ex, _ = experts(torch, 8, 256, 128)
    state = [routed(torch, T, 4, 8, 256, torch.bfloat16, seed=T) for T in (3, 900, 6000, 11000)]
    dys = [torch.randn_like(x) for x, _, _ in state]

    def step(i, stream=None):
        y, kept = ex.forward(*state[i], stream=stream, keep=True)
        return (y, *ex.backward(dys[i], kept, stream=stream))

    want = [step(i) for i in range(4)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for p, q in ((2, 3), (1, 2), (0, 3), (3, 1), (2, 2)):
        got = []
        for _ in range(3):
            got.append((p, step(p, a)))
            got.append((q, step(q, b)))
        torch.cuda.synchronize()
        for i, out in got:
            for x, y in zip(out, want[i]):
                assert torch.equal(x, y)
