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


class OnDevice:
    """Stands for a [rows][cols] tensor on a GPU of some index."""

    def __init__(self, dev, rows=3, cols=128, dtype=torch.bfloat16):
        self.dev, self.shape, self.dtype = dev, (rows, cols) if cols else (rows,), dtype

    def get_device(self):
        return self.dev

    def is_contiguous(self):
        return True

    def __getitem__(self, rows):
        return self


def test_host_tensors(world):
    """The stages take addresses: a host one would reach the GPU."""
    L, moe, layer, calls, rows, routing = world
    host = rows.clone()
    gpu = OnDevice(0)
    for kw in (dict(x=host, y=host, ws=host), dict(x=gpu, y=host, ws=gpu),
               dict(x=gpu, y=gpu, ws=host), dict(x=gpu, y=OnDevice(1), ws=gpu),
               dict(x=gpu, y=gpu, ws=OnDevice(1)), dict(x=gpu, y=gpu, ws=gpu, shared=host),
               dict(x=gpu, y=gpu, ws=gpu, resid=OnDevice(1))):
        with pytest.raises(L.MoeError):
            layer.forward_scored(routing=routing, **kw)
        assert calls == [], kw


def test_routing_and_bias_are_checked_first(world):
    L, moe, layer, calls, rows, routing = world
    gpu = OnDevice(0)
    for bad in (dict(n_groups=3), dict(score=7), dict(scale=float("nan")), dict(top_groups=2)):
        r = L.Routing.from_buffer_copy(routing)
        for name, v in bad.items():
            setattr(r, name, v)
        with pytest.raises(L.MoeError):
            layer.forward_scored(gpu, gpu, gpu, r)
        assert calls == [], bad
    for bias in (torch.zeros(8), OnDevice(1, 8, 0, torch.float32), OnDevice(0, 7, 0, torch.float32),
                 OnDevice(0, 8, 0)):
        with pytest.raises(L.MoeError):
            layer.forward_scored(gpu, gpu, gpu, routing, bias)
        assert calls == []


def test_runs_on_the_tensors_device(world, monkeypatch):
    """Every stage goes to the current stream of the device that x is on, whichever is
    the current one."""
    L, moe, layer, calls, rows, routing = world

    @contextlib.contextmanager
    def device(dev):
        calls.append(dev)
        yield
        calls.append("left")

    monkeypatch.setattr(torch.cuda, "device", device)
    x = OnDevice(1)
    assert layer.forward_scored(x, x, x, routing) is x
    assert calls == [1, "route", "route_scored", "experts", "combine", "left"]
