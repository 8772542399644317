"""MoeLayer.forward_scored refuses what it cannot run before it enqueues anything.
CPU only: the layer's stages are replaced by ones that record their calls."""
import contextlib

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def world(monkeypatch):
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    calls = []
    layer = moe.MoeLayer.__new__(moe.MoeLayer)
    layer.shape = L.Shape(128, 8, 2, 128, 128, 128, L.SCALE_BF16, L.PRECISION_W4A16)
    layer.device = "cpu"

    def stage(name, result):
        def call(*a, **k):
            calls.append(name)
            return result
        return call

    o = torch.zeros(3 * 2 + 3, 128, dtype=torch.bfloat16)
    monkeypatch.setattr(moe.MoeLayer, "route", stage("route", (torch.zeros(3, 2), None, None, None)))
    monkeypatch.setattr(moe.MoeLayer, "experts", stage("experts", o))
    monkeypatch.setattr(moe.MoeLayer, "combine", stage("combine", None))
    monkeypatch.setattr(moe, "route_scored", stage("route_scored", None))
    monkeypatch.setattr(moe, "_on", lambda stream: contextlib.nullcontext())
    rows = torch.zeros(3, 128, dtype=torch.bfloat16)
    routing = L.Routing(8, 2, L.SCORE_SIGMOID, 1, 1, L.GROUP_MAX, 1, 1.0)
    return L, moe, layer, calls, rows, routing


def test_w4a8_layer(world):
    """The expert stage has no W4A8 form; said before the router runs."""
    L, moe, layer, calls, rows, routing = world
    layer.shape.precision = L.PRECISION_W4A8
    with pytest.raises(L.MoeError, match="W4A16"):
        layer.forward_scored(rows, rows.clone(), None, routing)
    assert calls == []
