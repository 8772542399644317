"""Every form of the 8-bit product (tiles of 128, 96 and 64 rows, the split form's four) at what
happens next to a row: NaN among rows that share a stage of LDS, neighbouring columns of a
pitched y, offsets outside [0, N], capture, and one busy expert among hundreds without rows.  Each
call is checked to reach its form.  Bounds: test_gpu_fp8.py's."""
import pytest

import fp8_forms as F
import fp8_reference as R
from test_gpu_fp8 import check, gen, state, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu

K = 272
EACH = pytest.mark.parametrize("call", F.CALLS, ids=F.name)


def inputs(torch, call, extra=5):  # noqa: F811
    dtype, _, counts, M = call
    F.reached(call, K, extra)
    print(f"[case] form {F.name(call)}", flush=True)
    return (*state(torch, counts, M, K, M, pad=(16, 0), extra=extra), getattr(torch, dtype))


@EACH
def test_pitched_outputs_at_odd_elements(torch, call):  # noqa: F811
    q, sq, w, scales, offsets, dt = inputs(torch, call)
    n, M = len(q), w.shape[1]
    q.as_strided((n, K + 16), (K + 16, 1)).view(torch.uint8)[:, K:] = 0x7F  # NaN between the rows
    for before, behind in ((1, 2), (3, 0), (0, 5)):
        buf = torch.full((n, M + before + behind), 3.0, device="cuda", dtype=dt)
        check(torch, q, sq, w, scales, offsets, dt, y=buf[:, before:before + M])
        assert (buf[:, :before] == 3).all() and (buf[:, before + M:] == 3).all()
        assert (buf[int(offsets[-1]):] == 3).all()


@EACH
def test_nan_stays_in_its_row_and_column(torch, call):  # noqa: F811
    from ainfer_amd import moe
    q, sq, w, scales, offsets, dt = inputs(torch, call)
    n, M = len(q), w.shape[1]
    live = int(offsets[-1])

    def run(q, sq, w, scales):
        return moe.Fp8Weights(w, scales).product(q, sq, torch.zeros(n, M, device="cuda", dtype=dt), offsets)

    want = run(q, sq, w, scales)
    assert want.isfinite().all()
    rows = sorted({1, min(37, live - 1), live // 2, live - 1})
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[rows] = False
    for codes in (True, False):  # a code, a scale
        bad, bad_s = q.clone(), sq.clone()
        for i, r in enumerate(rows):
            if codes:
                bad.view(torch.uint8)[r, (97 * i + 5) % K] = 0xFF
            else:
                bad_s[r, i % 3] = float("nan")
        got = run(bad, bad_s, w, scales)
        assert got[rows].isnan().all() and torch.equal(got[keep], want[keep])
    # a weight of the first expert: its column of that expert's rows
    first = int(offsets[1])
    bad = w.clone()
    columns = sorted({0, 21, M // 2, M - 1})
    for i, m in enumerate(columns):
        bad.view(torch.uint8)[0, m, (130 * i + 3) % K] = 0x7F
    got = run(q, sq, bad, scales)
    assert got[:first, columns].isnan().all()
    got[:first, columns] = want[:first, columns]
    assert torch.equal(got, want)
    # a block's scale: its 128 columns
    bad = scales.clone()
    block = scales.shape[1] - 1
    bad[0, block, 1] = float("nan")
    got = run(q, sq, w, bad)
    assert got[:first, 128 * block:].isnan().all()
    got[:first, 128 * block:] = want[:first, 128 * block:]
    assert torch.equal(got, want)


@EACH
def test_offsets_out_of_range(torch, call):  # noqa: F811
    """They are the ends of [0, N]; rows on both sides of y stay."""
    from ainfer_amd import moe
    q, sq, w, scales, offsets, dt = inputs(torch, call, extra=0)
    n, M = len(q), w.shape[1]
    buf = torch.full((n + 20, M), 4.0, device="cuda", dtype=dt)
    wide = offsets.clone()
    wide[0], wide[-1] = -7, 1 << 30
    moe.Fp8Weights(w, scales).product(q, sq, buf[10:-10], wide)
    assert (buf[:10] == 4).all() and (buf[-10:] == 4).all()
    assert torch.equal(buf[10:-10], moe.Fp8Weights(w, scales, dt).product(q, sq, offsets=offsets))


@EACH
def test_captured(torch, call):  # noqa: F811
    """Replays on other codes and other offsets equal eager calls; on another stream too."""
    from ainfer_amd import moe
    q, sq, w, scales, offsets, dt = inputs(torch, call)
    f = moe.Fp8Weights(w, scales, dt)
    n, M = len(q), w.shape[1]
    y = torch.zeros(n, M, device="cuda", dtype=dt)
    f.product(q, sq, y, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f.product(q, sq, y, offsets)
    s = torch.cuda.Stream()
    for i in range(4):
        q.copy_(R.codes(gen(torch, 50 + i), *q.shape))
        if len(offsets) > 2:
            offsets[1:-1] = (91 * i + 3) % n
        y.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.full_like(y, i)
        s.wait_stream(torch.cuda.current_stream())
        f.product(q, sq, want, offsets, stream=s)
        s.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("call", F.BUSY, ids=F.name)
def test_one_busy_expert(torch, call):  # noqa: F811
    q, sq, w, scales, offsets, dt = inputs(torch, call)
    y = check(torch, q, sq, w, scales, offsets, dt)
    again = torch.full_like(y, 3)
    from ainfer_amd import moe
    moe.Fp8Weights(w, scales).product(q, sq, again, offsets)
    n = int(offsets[-1])
    assert torch.equal(again[:n], y[:n]) and (again[n:] == 3).all()
