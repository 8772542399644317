"""A step with the residual stream added in it: y = x + experts(x), and its gradient.

Bounds.  In fp32 the sum of the experts' rows and the residual is rounded once, as their sum
is when it is taken of two fp32 tensors: the same bits.  In bf16 the sum of fp32 values is
rounded once, by 2^-8 of it at most, and dx without the residual once, by 2^-8 of it (2^-7
together, with the fp32 roundings beside).  Against 64 bits: test_gpu_fp8_experts.py's 0.14 of
the experts' share."""
import pytest

from test_gpu_fp8_experts import experts, routed, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("T,k,E,H,I", ((1, 4, 8, 256, 128), (40, 4, 16, 272, 144), (500, 2, 4, 512, 256)))
def test_gradient_with_the_residual(torch, T, k, E, H, I, dtype):  # noqa: F811
    dt = getattr(torch, dtype)
    ex, (gu, dn) = experts(torch, E, H, I, y_dtype=torch.float32)
    x, idx, w = routed(torch, T, k, E, H, dt)
    idx[::3, 0] = -1
    dy = torch.randn(T, H, device="cuda").to(dt)
    _, kept = ex.forward(x, idx, w, resid=x, keep=True)
    dx, dw = ex.backward(dy, kept, resid=dy)
    share, dw0 = ex.backward(dy, kept)
    assert torch.equal(dw, dw0)
    if dt == torch.float32:
        assert torch.equal(dx, share + dy)
    else:
        want = share.double() + dy.double()
        assert ((dx.double() - want).abs() <= 2.0 ** -7 * (share.double().abs() + want.abs())).all()
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    h, _, _, pos, _ = kept
    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if len(t):
            he = h.double()[pos[t, j].long()].requires_grad_()
            a = torch.nn.functional.silu(he[:, :I]) * he[:, I:]
            a.backward((w[t, j].double()[:, None] * dy[t].double()) @ dn[e])
            ref.index_add_(0, t, he.grad @ gu[e])
    off = (dx.double() - (ref + dy.double())).norm()
    assert off <= 0.14 * ref.norm() + 2.0 ** -8 * (ref + dy.double()).norm()


def test_captured(torch):  # noqa: F811
    ex, _ = experts(torch, 8, 256, 128)
    x, idx, w = routed(torch, 30, 3, 8, 256, torch.bfloat16)
    dy = torch.randn(30, 256, device="cuda").to(torch.bfloat16)

    def step():
        y, kept = ex.forward(x, idx, w, resid=x, keep=True)
        return (y, *ex.backward(dy, kept, resid=dy))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for t, n in zip((x, idx, w), routed(torch, 30, 3, 8, 256, torch.bfloat16, seed=10 + i)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_refusals(torch):  # noqa: F811
    from ainfer_amd import _lib as L
    ex, _ = experts(torch, 4, 256, 128)
    x, idx, w = routed(torch, 5, 2, 4, 256, torch.bfloat16)
    _, kept = ex.forward(x, idx, w, resid=x, keep=True)
    for bad in (x[:4], x.float(), x.cpu(), x[:, :240], x[0], x.t().contiguous().t()):
        with pytest.raises(L.MoeError):
            ex.backward(x, kept, resid=bad)
