"""Token sorts at the border between the launch that counts all pairs by itself and the two that share
their counts (3 rounds of 16384 pairs): places and offsets are the definition's on both sides."""
import pytest

import fp8_reference as R
from test_gpu_sort import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ("even", "one", "power", "dropped"))
@pytest.mark.parametrize("E", (1, 16, 1000))
@pytest.mark.parametrize("T,k", ((49151, 1), (6144, 8), (49153, 1), (4915, 10), (4916, 10), (32768, 1), (32769, 1)))
def test_border(torch, T, k, E, kind):  # noqa: F811
    from ainfer_amd import moe
    print(f"[case] sort {T} {k} {E} {kind}", flush=True)
    g = torch.Generator()
    g.manual_seed(T + E)
    if kind == "one":
        idx = torch.full((T, k), E // 2)
    elif kind == "power":
        idx = (E * torch.rand(T, k, generator=g) ** 3).long().clamp_max(E - 1)
    else:
        most = E if kind == "even" else 2 * E + 1
        idx = torch.randint(0, most, (T, k), generator=g) - (0 if kind == "even" else E // 2 + 1)
    idx = idx.int().cuda()
    x = torch.randn(T, 8, device="cuda")
    rows, _, offsets, pos = moe.sort_rows(x, idx, E, moe.sort_workspace(T, k, E))
    woff, wpos, order = R.sort(idx, E)
    assert torch.equal(offsets.cpu(), woff) and torch.equal(pos.cpu(), wpos)
    assert torch.equal(rows[:len(order)], x[torch.tensor(order, device="cuda", dtype=torch.long) // k])
