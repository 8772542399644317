"""The gated activation (ainfer_moe_silu_mul) against its formula in 64 bits.

Bound: exp to 2^-22 of itself (its argument's rounding included for |g| <= 16, and
g / (1 + exp(-g)) moves by less than exp does), one addition, one division and one
product of 2^-24 each: 2^-21 relative in fp32; bf16 rounds once more (2^-8)."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def expected(g, u):
    g, u = g.double(), u.double()
    return g / (1 + (-g).exp()) * u


def check(torch, g, u, act):
    from ainfer_amd import moe
    print(f"[case] {tuple(g.shape)} {g.dtype} -> {act.dtype} pitches {g.stride(0)} {u.stride(0)} "
          f"{act.stride(0)}", flush=True)
    want = expected(g, u)
    moe.silu_mul(g, u, act)
    torch.cuda.synchronize()
    rel = 2.0 ** -21 + (2.0 ** -8 if act.dtype == torch.bfloat16 else 0)
    assert ((act.double() - want).abs() <= rel * want.abs() + 1e-37).all()


DTYPES = (("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"),
          ("bfloat16", "float32"))


@pytest.mark.parametrize("di,do", DTYPES)
@pytest.mark.parametrize("T,I", ((1, 1), (1, 7), (3, 8), (5, 1024), (17, 883), (64, 512),
                                 (300, 130), (2, 17408)))
def test_matches_formula(torch, di, do, T, I):
    g = torch.randn(T, I, device="cuda").mul_(2).to(getattr(torch, di))
    u = torch.randn(T, I, device="cuda").to(getattr(torch, di))
    check(torch, g, u, torch.empty(T, I, device="cuda", dtype=getattr(torch, do)))


@pytest.mark.parametrize("di,do", DTYPES)
def test_pitches(torch, di, do):
    """gate and up as the halves of one buffer, aligned and not; a wider act
    whose other columns stay as they were."""
    for I, pad in ((64, 8), (64, 1), (50, 6), (7, 0)):
        gu = torch.randn(9, 2 * I + pad, device="cuda").to(getattr(torch, di))
        wide = torch.full((9, I + 3), 7.0, device="cuda", dtype=getattr(torch, do))
        check(torch, gu[:, :I], gu[:, I:2 * I], wide[:, :I])
        assert (wide[:, I:] == 7).all()
        act = torch.empty(9, I, device="cuda", dtype=getattr(torch, do))
        check(torch, gu[:, :I], gu[:, I:2 * I], act)


def test_in_place(torch):
    for dt in (torch.float32, torch.bfloat16):
        for which in (0, 1):
            gu = [torch.randn(20, 100, device="cuda").to(dt) for _ in range(2)]
            want = expected(*gu)
            from ainfer_amd import moe
            moe.silu_mul(gu[0], gu[1], gu[which])
            rel = 2.0 ** -21 + (2.0 ** -8 if dt == torch.bfloat16 else 0)
            assert ((gu[which].double() - want).abs() <= rel * want.abs() + 1e-37).all()


def test_large_and_special_values(torch):
    from ainfer_amd import moe
    g = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -0.0, 100.0, -100.0, 3e38, -3e38]],
                     device="cuda")
    u = torch.ones_like(g)
    act = torch.empty_like(g)
    moe.silu_mul(g, u, act)
    a = act[0].tolist()
    assert a[0] == math.inf and math.isnan(a[1]) and math.isnan(a[2])
    assert a[3] == 0 and a[4] == 0 and a[5] == 100.0 and abs(a[6]) < 1e-37
    assert a[7] == g[0, 7].item() and a[8] == 0


def test_graph_and_large_rows(torch):
    from ainfer_amd import moe
    g = torch.randn(70, 333, device="cuda")
    u = torch.randn(70, 333, device="cuda")
    act = torch.empty_like(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.silu_mul(g, u, act)
    for _ in range(3):
        g.normal_()
        act.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(g)
        moe.silu_mul(g, u, eager)
        assert torch.equal(act, eager)
    # 2^31 elements and more
    T, I = 65536, 33000
    g = torch.empty(T, I, device="cuda", dtype=torch.bfloat16)
    u = torch.ones_like(g)
    for t in range(0, T, 8192):
        g[t:t + 8192].normal_()
    act = torch.empty_like(g)
    moe.silu_mul(g, u, act)
    torch.cuda.synchronize()
    for t in (0, 40000, 65535):
        want = expected(g[t], u[t])
        assert ((act[t].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want.abs() + 1e-37).all()
