"""Tokens sorted by expert and back, with weights and gradients, against plain forms.

Bounds.  Sorting and copies are exact.  Weighted sums: k products and additions in
fp32, each off by 2^-24 of the sum of magnitudes; gradients of weights: sums of H
products, (H + 8) 2^-24 of the sum of magnitudes; outputs are rounded once (bf16 2^-8)."""
import pytest

import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def ids(torch, T, k, E, seed, kind="any"):
    g = gen(torch, seed)
    if kind == "one":
        return torch.full((T, k), E - 1, dtype=torch.int32, device="cuda")
    if kind == "none":
        return torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    lo, hi = (-(E // 2) - 1, E + E // 2 + 2) if kind == "dropped" else (0, E)
    return torch.randint(lo, hi, (T, k), generator=g, device="cuda", dtype=torch.int32)


SIZES = ((1, 1, 1), (1, 8, 256), (2, 3, 5), (7, 32, 1024), (64, 8, 64), (129, 10, 512), (300, 6, 96),
         (1003, 7, 1024), (2048, 1, 7), (2049, 1, 7), (1024, 8, 64), (1025, 8, 64), (4096, 8, 64),
         (5000, 32, 33), (8193, 32, 100), (16385, 17, 3), (2560, 16, 600), (2731, 15, 1024),
         (4099, 10, 8))


@pytest.mark.parametrize("kind", ("any", "dropped", "one", "none"))
@pytest.mark.parametrize("T,k,E", SIZES)
def test_sort(torch, T, k, E, kind):
    """Copies of bf16 rows; rows of dropped pairs, and columns between rows, stay."""
    from ainfer_amd import moe
    print(f"[case] sort {T} {k} {E} {kind}", flush=True)
    idx = ids(torch, T, k, E, T + k, kind)
    H = 40
    x = torch.randn(T, H, generator=gen(torch, 1), device="cuda").to(torch.bfloat16)
    offsets, pos, order = R.sort(idx, E)
    buf = torch.full((T * k + 2, H + 3), 5.0, device="cuda", dtype=torch.bfloat16)
    out = (buf[1:T * k + 1, 1:H + 1], None, torch.empty(E + 1, dtype=torch.int32, device="cuda"),
           torch.empty(T, k, dtype=torch.int32, device="cuda"))
    moe.sort_rows(x, idx, E, moe.sort_workspace(T, k, E), out=out)
    assert torch.equal(out[2].cpu(), offsets) and torch.equal(out[3].cpu(), pos)
    want = torch.full_like(buf, 5.0)
    if order:
        want[1:len(order) + 1, 1:H + 1] = x[torch.tensor(order, device="cuda") // k]
    assert torch.equal(buf, want)


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("H", (1, 3, 5, 7, 8, 9, 15, 130, 515, 2047, 4096))
def test_sort_row_lengths(torch, H, dtype):
    from ainfer_amd import moe
    dt = getattr(torch, dtype)
    for T, k, E in ((3, 4, 8), (700, 4, 8)):
        idx = ids(torch, T, k, E, H, "dropped")
        x = torch.randn(T, H + 5, generator=gen(torch, H), device="cuda").to(dt)[:, 2:H + 2]
        rows, sc, offsets, pos = moe.sort_rows(x, idx, E, moe.sort_workspace(T, k, E))
        woff, wpos, order = R.sort(idx, E)
        assert sc is None and torch.equal(offsets.cpu(), woff) and torch.equal(pos.cpu(), wpos)
        assert torch.equal(rows[:len(order)], x[torch.tensor(order, device="cuda") // k])


@pytest.mark.parametrize("pow2", (False, True))
@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("T,k,E,H", ((1, 8, 256, 4096), (1, 1, 1, 16), (5, 3, 7, 144), (40, 10, 512, 2048),
                                     (333, 8, 60, 272), (2000, 4, 16, 1040)))
def test_sort_quantised(torch, T, k, E, H, dtype, pow2):
    """The sorted codes and scales are the token rows' own."""
    from ainfer_amd import moe
    print(f"[case] sort fp8 {T} {k} {E} {H} {dtype} {pow2}", flush=True)
    idx = ids(torch, T, k, E, T, "dropped")
    x = torch.randn(T, H, generator=gen(torch, T + H), device="cuda").to(getattr(torch, dtype))
    q = torch.full((T * k, H + 16), 2.0, device="cuda").to(R.E4M3)
    s = torch.full((T * k, R.groups(H)), -1.0, device="cuda")
    off, pos = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((E + 1,), (T, k)))
    moe.sort_rows(x, idx, E, moe.sort_workspace(T, k, E), pow2=pow2, out=(q[:, :H], s, off, pos))
    woff, wpos, order = R.sort(idx, E)
    assert torch.equal(off.cpu(), woff) and torch.equal(pos.cpu(), wpos)
    wq, ws = R.quantised(x, pow2)
    n, tok = len(order), torch.tensor(order, dtype=torch.int64) // k
    assert torch.equal(q[:n, :H].cpu().view(torch.uint8), wq[tok].view(torch.uint8))
    assert torch.equal(s[:n].cpu(), ws[tok])
    assert (q[n:].float() == 2).all() and (q[:, H:].float() == 2).all() and (s[n:] == -1).all()


def test_sort_no_tokens(torch):
    from ainfer_amd import moe
    x = torch.empty(0, 64, device="cuda")
    off = torch.full((9,), 7, dtype=torch.int32, device="cuda")
    idx = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    moe.sort_rows(x, idx, 8, moe.sort_workspace(0, 2, 8), out=(x, None, off, idx.clone()))
    assert (off == 0).all()


def test_sort_places_alone(torch):
    """Without rows: offsets and places, through the C entry."""
    import ctypes as C
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    for T, k, E in ((3, 4, 8), (600, 4, 8), (5000, 4, 8)):
        idx = ids(torch, T, k, E, T, "dropped")
        ws = moe.sort_workspace(T, k, E)
        off, pos = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((E + 1,), (T, k)))
        d = L.Sorting(E, k, 64, L.ACT_BF16, 0, 0)
        L.check(L.lib().ainfer_moe_sort_rows(
            C.byref(d), None, 0, idx.data_ptr(), T, off.data_ptr(), pos.data_ptr(), None, 0, None,
            ws.data_ptr(), ws.nbytes, torch.cuda.current_stream().cuda_stream))
        woff, wpos, _ = R.sort(idx, E)
        assert torch.equal(off.cpu(), woff) and torch.equal(pos.cpu(), wpos)


def test_sort_largest(torch):
    """65536 tokens of 32 experts each: rows of more than 2^31 elements."""
    from ainfer_amd import moe
    T, k, E, H = 65536, 32, 1000, 1040
    idx = ids(torch, T, k, E, 4, "dropped")
    x = torch.randn(T, H, generator=gen(torch, 2), device="cuda").to(torch.bfloat16)
    rows, _, offsets, pos = moe.sort_rows(x, idx, E, moe.sort_workspace(T, k, E))
    key = idx.flatten().long()
    key = torch.where((key >= 0) & (key < E), key, E)
    in_order, order = torch.sort(key, stable=True)
    woff = torch.searchsorted(in_order, torch.arange(E + 1, device="cuda"))
    assert torch.equal(offsets.long(), woff)
    n = int(woff[-1])
    assert torch.equal(pos.flatten()[order[:n]].long(), torch.arange(n, device="cuda"))
    assert (pos.flatten()[order[n:]] == -1).all()
    for a in range(0, n, 1 << 18):
        b = min(n, a + (1 << 18))
        assert torch.equal(rows[a:b], x[order[a:b] // k])
    # and back: every token's rows are the token, weights of 1 / (kept pairs)
    kept = (pos >= 0).sum(1, keepdim=True).clamp_min(1)
    y = moe.unpermute(rows, pos, (1.0 / kept).float().expand(T, k).contiguous(), torch.empty_like(x))
    assert ((y.double() - x.double()).abs() <= (2.0 ** -8 + 34 * 2.0 ** -24) * x.double().abs()).all()


# ---- back -------------------------------------------------------------------------

def back_state(torch, T, k, E, H, rows_dtype, y_dtype, pad=0, seed=0, kind="dropped"):
    g = gen(torch, seed + T + H)
    pos = R.sort(ids(torch, T, k, E, seed, kind), E)[1].cuda()
    dts = getattr(torch, rows_dtype), getattr(torch, y_dtype)
    rows = torch.randn(T * k, H + pad, generator=g, device="cuda").to(dts[0])[:, pad // 2:pad // 2 + H]
    w = torch.rand(T, k, generator=g, device="cuda") - 0.2
    dy = torch.randn(T, H + pad, generator=g, device="cuda").to(dts[1])[:, :H]
    return pos, rows, w, dy


DTYPES = (("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float32", "bfloat16"),
          ("float32", "float32"))
BACK = ((1, 1, 1, 1), (1, 8, 64, 4096), (3, 2, 5, 7), (16, 8, 256, 2048), (50, 10, 32, 515), (333, 32, 64, 64),
        (1030, 3, 16, 1000), (5, 3, 4, 9), (40, 6, 8, 2055))


def half_step(torch, dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24


@pytest.mark.parametrize("rd,yd", DTYPES)
@pytest.mark.parametrize("T,k,E,H", BACK)
def test_unpermute(torch, T, k, E, H, rd, yd):
    from ainfer_amd import moe
    print(f"[case] unpermute {T} {k} {H} {rd} {yd}", flush=True)
    for pad in (0, 3):
        pos, rows, w, resid = back_state(torch, T, k, E, H, rd, yd, pad)
        there = (pos >= 0)
        mine = rows.double()[pos.clamp_min(0).long()]
        for weights in (w, None):
            for res in (None, resid):
                f = torch.where(there, w.double() if weights is not None else 1.0, 0.0)
                terms = f[:, :, None] * mine
                want, size = terms.sum(1), terms.abs().sum(1)
                if res is not None:
                    want, size = want + res.double(), size + res.double().abs()
                buf = torch.full((T, H + 2), 8.0, device="cuda", dtype=resid.dtype)
                y = buf[:, 1:H + 1]
                moe.unpermute(rows, pos, weights, y, resid=res)
                bound = (k + 2) * 2.0 ** -24 * size * 1.01 + half_step(torch, y.dtype) * want.abs()
                assert ((y.double() - want).abs() <= bound).all()
                assert (buf[:, 0] == 8).all() and (buf[:, -1] == 8).all()


@pytest.mark.parametrize("H", (136, 137, 143, 9, 5))
def test_unpermute_over_its_residual_and_bad_places(torch, H):
    """resid as y; places outside the rows are left out, NaN weights of theirs too."""
    from ainfer_amd import moe
    pos, rows, w, resid = back_state(torch, 40, 4, 8, H, "float32", "float32", kind="any")
    y = moe.unpermute(rows, pos, w, torch.empty_like(resid), resid=resid)
    z = resid.clone()
    moe.unpermute(rows, pos, w, z, resid=z)
    assert torch.equal(y, z)
    bad, wb = pos.clone(), w.clone()
    bad[::2, 1], bad[1::2, 2] = 160, -7
    bad[3, 3] = 1 << 30
    gone = (bad < 0) | (bad >= 160)
    wb[gone] = float("nan")
    wz = torch.where(gone, 0.0, w)
    a = moe.unpermute(rows, bad, wb, torch.empty_like(y))
    b = moe.unpermute(rows, pos, wz, torch.empty_like(y))
    assert torch.equal(a, b)
    dr, dw = (torch.full_like(rows, 6.0), torch.empty_like(w))
    moe.unpermute_backward(resid, rows, bad, wb, dr, dw)
    assert (dw[gone] == 0).all()
    lost = pos[gone].long()
    assert (dr[lost] == 6).all() and dr.isfinite().all()


@pytest.mark.parametrize("rd,yd", DTYPES)
@pytest.mark.parametrize("T,k,E,H", BACK)
def test_unpermute_backward(torch, T, k, E, H, rd, yd):
    """Against the formulas, and drows and dw as the slopes of <dy, y> (y is linear in
    both, so a difference is a slope)."""
    from ainfer_amd import moe
    print(f"[case] backward {T} {k} {H} {rd} {yd}", flush=True)
    for pad in (0, 3):
        pos, rows, w, dy = back_state(torch, T, k, E, H, rd, yd, pad)
        there = pos >= 0
        at = pos.clamp_min(0).long()
        drows = torch.full((T * k, H + pad), 4.0, device="cuda", dtype=rows.dtype)[:, pad:]
        dw = torch.empty_like(w)
        moe.unpermute_backward(dy, rows, pos, w, drows, dw)
        terms = dy.double()[:, None, :] * rows.double()[at]
        want = torch.where(there, terms.sum(2), 0.0)
        size = torch.where(there, terms.abs().sum(2), 0.0)
        assert ((dw.double() - want).abs() <= (H + 8) * 2.0 ** -24 * size).all()
        wr = (w.double()[:, :, None] * dy.double()[:, None, :])[there]
        got = drows.double()[pos[there].long()]
        assert ((got - wr).abs() <= (2.0 ** -24 + half_step(torch, rows.dtype)) * wr.abs() * 1.01).all()
        n = int(there.sum())
        assert (drows[n:] == 4).all()
        # one of the two alone: the same values
        d2, w2 = torch.full_like(drows, 4.0), torch.empty_like(w)
        moe.unpermute_backward(dy, rows, pos, w, drows=d2)
        moe.unpermute_backward(dy, rows, pos, w, dw=w2)
        assert torch.equal(d2, drows) and torch.equal(w2, dw)
        moe.unpermute_backward(dy, rows, pos, None, drows=d2)
        assert torch.equal(d2[pos[there].long()],
                           dy[:, None, :].expand(T, k, H)[there].to(d2.dtype))
        # differences
        step = torch.randn(T, k, generator=gen(torch, 9), device="cuda")
        y0 = moe.unpermute(rows, pos, w, torch.empty(T, H, device="cuda"))
        y1 = moe.unpermute(rows, pos, w + step, torch.empty(T, H, device="cuda"))
        rise = (dy.double() * (y1.double() - y0.double())).sum()
        scale = (dy.double().abs()[:, None, :] * rows.double().abs()[at]
                 * (w.double().abs() + (w + step).double().abs())[:, :, None] * there[:, :, None]).sum()
        assert abs(rise - (dw.double() * step.double()).sum()) <= (H + 3 * k + 20) * 2.0 ** -24 * scale


def test_sort_then_back_is_the_gradient(torch):
    """<rows' gradient, sort_rows(v)> = <unpermute of it, v> for every v."""
    from ainfer_amd import moe
    T, k, E, H = 200, 5, 12, 72
    idx = ids(torch, T, k, E, 6, "dropped")
    ws = moe.sort_workspace(T, k, E)
    v = torch.randint(-3, 4, (T, H), device="cuda").float()
    rows = torch.zeros(T * k, H, device="cuda")
    off, pos = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((E + 1,), (T, k)))
    moe.sort_rows(v, idx, E, ws, out=(rows, None, off, pos))
    d = torch.randint(-3, 4, (T * k, H), device="cuda").float()
    dx = moe.unpermute(d, pos, None, torch.empty_like(v))
    assert (d.double() * rows.double()).sum() == (dx.double() * v.double()).sum()  # whole numbers


def test_streams_graphs(torch):
    """Captured once, replayed on other ids and rows with eager work between; two
    captured calls share a workspace."""
    from ainfer_amd import moe
    for T, k, E, H in ((2, 4, 16, 256), (900, 4, 16, 272)):
        ws = moe.sort_workspace(T, k, E)
        x = torch.randn(T, H, generator=gen(torch, 1), device="cuda")
        idx = ids(torch, T, k, E, 1, "dropped")
        w = torch.rand(T, k, device="cuda")

        def call():
            a = moe.sort_rows(x, idx, E, ws, fp8=True)
            b = moe.sort_rows(x, idx, E, ws)
            y = moe.unpermute(b[0], b[3], w, torch.empty_like(x))
            return [*a, b[0], b[2], b[3], y]

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for i in range(4):
            x.normal_(generator=gen(torch, 50 + i))
            idx.copy_(ids(torch, T, k, E, 60 + i, "dropped"))
            graph.replay()
            torch.cuda.synchronize()
            want = call()
            n = int(want[2][-1])
            for g, u in zip(got, want):
                m = n if g.shape[0] == T * k else len(g)
                assert torch.equal(g[:m].view(torch.uint8), u[:m].view(torch.uint8))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        rows, _, off, pos = moe.sort_rows(x, idx, E, ws, stream=s)
        y = moe.unpermute(rows, pos, w, torch.empty_like(x), stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(off, want[5]) and torch.equal(y, want[7])
