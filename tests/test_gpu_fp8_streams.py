"""Weights laid out on a stream of their own: the codes may be dropped at once."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.mark.parametrize("transpose", (False, True))
def test_codes_dropped_while_the_stream_is_busy(torch, transpose):
    """Their memory, and that of scales that are laid out anew, is not given out while the
    stream has not come to them."""
    from ainfer_amd import moe
    w = torch.randint(0, 256, (2, 256, 512), device="cuda", dtype=torch.uint8)
    scales = torch.rand(2, 2, 4, device="cuda")
    f = moe.Fp8Weights(w, scales, transpose=transpose)
    want, want_scales = f.packed.clone(), f.scales.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)  # some tens of ms
    f = moe.Fp8Weights(w, scales, transpose=transpose, stream=s)
    taken = {t.data_ptr() for t in (w, scales)}
    del w, scales
    fresh = []
    for _ in range(4):
        fresh.append(torch.zeros(2, 256, 512, device="cuda", dtype=torch.uint8))
        fresh.append(torch.zeros(2, 2, 4, device="cuda"))
    assert not s.query()  # all of this came before the layout
    assert not taken & {t.data_ptr() for t in fresh}
    s.synchronize()
    assert torch.equal(f.packed, want) and torch.equal(f.scales, want_scales)
