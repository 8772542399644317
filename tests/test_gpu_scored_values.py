"""Scored routing (ainfer_moe_route_scored) on rows whose answer is written out by
hand, alone (a wave a token) and as many tokens (four a wave)."""
import math

import pytest

from test_gpu_scored import GMAX, GTOP2, RTOL, SIG, SOFT, torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
INF = math.inf


def check(torch, row, bias, k, score, want, G=1, top=1, gscore=GMAX, renorm=0, scale=1.0,
          dtype="float32", atol=0.0):
    """want: [(expert, weight)]"""
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    print(f"[case] {len(row)} experts k={k} score={score} G={G}/{top} {dtype} renorm={renorm}",
          flush=True)
    x = torch.tensor([row], device="cuda", dtype=getattr(torch, dtype))
    b = None if bias is None else torch.tensor(bias, device="cuda", dtype=torch.float32)
    r = L.Routing(len(row), k, score, G, top, gscore, renorm, scale)
    for T in (1, 5, 16385):
        idx, w = moe.route_scored(r, x.expand(T, -1).contiguous(), b)
        assert idx.cpu().tolist() == [[e for e, _ in want]] * T
        exact = torch.tensor([[v for _, v in want]], dtype=torch.float64)
        assert ((w.cpu().double() - exact).abs() <= RTOL * exact.abs() + atol).all()


def test_a_bias_selects_and_changes_no_score(torch):
    """softmax's sum holds the experts that only their bias masks: exp gives 3, 1, 4 of 8."""
    check(torch, [0.0, 0.0], [0.0, -INF], 1, SOFT, [(0, 0.5)])
    row = [math.log(3), 0.0, math.log(4)]
    for masked in (-INF, math.nan):
        check(torch, row, [0.0, 0.0, masked], 2, SOFT, [(0, 0.375), (1, 0.125)])
        # 0.375 and 0.125 + 0.3; over the first two alone 0.75 and 0.25 + 0.3
        check(torch, row, [0.0, 0.3, masked], 1, SOFT, [(1, 0.125)])
        check(torch, row, [0.0, 0.3, masked], 2, SOFT, [(1, 0.25), (0, 0.75)], renorm=1)
        check(torch, row, [0.0, 0.3, masked], 3, SOFT, [(1, 0.125), (0, 0.375), (2, 0.0)])
    # a masked logit is not in the sum
    check(torch, [0.0, 0.0, -INF], [0.0, 0.1, 9.0], 2, SOFT, [(1, 0.5), (0, 0.5)])
    # groups of 3.5 and 0.5, and of 4 and a masked 8, of 16: by the largest key 0.219
    # against 0.25 + 0.1, by the two largest 0.25 + 0.03 against 0.25
    row = [math.log(v) for v in (3.5, 0.5, 4.0, 8.0)]
    check(torch, row, [0.0, 0.0, 0.1, -INF], 1, SOFT, [(2, 0.25)], G=2, top=1)
    check(torch, row, [0.03, 0.0, 0.0, -INF], 1, SOFT, [(0, 0.21875)], G=2, top=1, gscore=GTOP2)


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
def test_an_infinite_logit_is_the_largest_of_its_type(torch, dtype):
    """It ties with the largest finite value, the lower index first."""
    most = torch.finfo(getattr(torch, dtype)).max
    for rest in (0, 5, 300):
        row = [most, INF, most] + [0.0] * rest
        for score, w in ((SOFT, 1 / 3), (SIG, 1.0)):
            check(torch, row, None, 2, score, [(0, w), (1, w)], dtype=dtype)
            check(torch, row, [0.0] * len(row), 2, score, [(0, w), (1, w)], dtype=dtype)
            check(torch, row[1:], None, 2, score, [(0, w if score == SIG else 1 / 2),
                                                   (1, w if score == SIG else 1 / 2)], dtype=dtype)


def test_scores_at_the_end_of_fp32(torch):
    """Not renormalised: full relative accuracy down to 2^-126, below it the weight may
    be 0 times scale, which is off by less than 2^-126 of it."""
    low = 2.0 ** -126

    def sig(l):
        return 1 / (1 + math.exp(-l))

    for scale in (1.0, 2.0 ** 100):
        check(torch, [-87.0, -86.5, -300.0, -80.0], None, 3, SIG,
              [(3, sig(-80.0) * scale), (1, sig(-86.5) * scale), (0, sig(-87.0) * scale)], scale=scale)
        check(torch, [-88.5, -90.0, -100.0, -88.0], None, 4, SIG,
              [(e, sig(l) * scale) for e, l in ((3, -88.0), (0, -88.5), (1, -90.0), (2, -100.0))],
              scale=scale, atol=low * scale)
        check(torch, [-87.0, 0.0, -40.0], None, 3, SOFT,
              [(1, scale), (2, math.exp(-40.0) * scale), (0, math.exp(-87.0) * scale)], scale=scale)
        check(torch, [-88.0, 0.0, -103.0], None, 3, SOFT,
              [(1, scale), (0, math.exp(-88.0) * scale), (2, math.exp(-103.0) * scale)],
              scale=scale, atol=low * scale)
    # renormalised, such scores keep their ratios
    check(torch, [-89.0, -90.0], None, 2, SIG, [(0, 1 / (1 + math.exp(-1))),
                                                (1, 1 / (1 + math.exp(1)))], renorm=1)
