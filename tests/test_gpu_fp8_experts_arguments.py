"""Experts in 8-bit floating point refuse a wrong tensor before the first kernel."""
import pytest

from test_gpu_fp8_experts import experts, routed, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def calls(monkeypatch):
    """The library's functions that were called."""
    from ainfer_amd import moe
    seen, call = [], moe._call

    def record(fn, *args):
        seen.append(fn.__name__)
        return call(fn, *args)

    monkeypatch.setattr(moe, "_call", record)
    return seen


def test_forward(torch, calls):  # noqa: F811
    from ainfer_amd import _lib as L
    ex, _ = experts(torch, 4, 256, 128)
    x, idx, w = routed(torch, 5, 2, 4, 256, torch.bfloat16)
    calls.clear()
    ex.forward(x, idx, w, y=torch.empty_like(x), resid=x)
    assert [n.removeprefix("ainfer_moe_") for n in calls] == [
        "sort_rows", "fp8_product", "silu_mul_fp8", "fp8_product", "unpermute"]
    calls.clear()
    f = torch.empty(5, 256, device="cuda")
    for kw in (dict(x=x[:4]), dict(x=x[:, :240]), dict(x=x.half()), dict(x=x.cpu()), dict(x=x[0]),
               dict(x=x.t().contiguous().t()), dict(idx=idx[:4]), dict(idx=idx.long()), dict(idx=idx[0]),
               dict(idx=idx.cpu()), dict(idx=idx.t().contiguous().t()), dict(w=w[:4]), dict(w=w[:, :1].contiguous()),
               dict(w=w.double()), dict(w=w.to(torch.bfloat16)), dict(w=w.cpu()), dict(w=w[0]),
               dict(w=w.t().contiguous().t()), dict(y=x[:4]), dict(y=f[:, :255]), dict(y=f.double()),
               dict(y=f.cpu()), dict(y=f.t().contiguous().t()), dict(y=f[0]), dict(resid=x[:4]),
               dict(resid=f), dict(y=f, resid=x), dict(resid=x.cpu()), dict(resid=x[:, :240])):
        args = dict(x=x, idx=idx, w=w)
        args.update(kw)
        with pytest.raises(L.MoeError):
            ex.forward(**args)
        assert not calls, kw
