"""The operators around the expert stage check every operand by itself: each has an
address of its own here, and one call differs from a valid one in one thing.  CPU
only: no call here reaches a kernel."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    from ainfer_amd import _lib
    return _lib


def at(n):
    """Operand n of a call: 1 GiB apart, 256-byte aligned."""
    return n << 30


LOGITS, BIAS, IDX, W = (at(n) for n in range(1, 5))


def route(L, logits=LOGITS, dtype=0, ld=256, bias=BIAS, T=4, idx=IDX, w=W, **kw):
    d = dict(n_experts=256, top_k=8, score=L.SCORE_SIGMOID, n_groups=8, top_groups=4,
             group_score=L.GROUP_TOP2, renormalize=1, scale=2.5)
    d.update(kw)
    return L.lib().ainfer_moe_route_scored(C.byref(L.Routing(**d)), logits, dtype, ld, bias, T,
                                           idx, w, None)


X, IDS, WS, Y0, Y1, A0, A1, B0, B1, RANKS, SCALES = (at(n) for n in range(11, 22))


def struct(L, a=(A0, A1), b=(B0, B1), out=(100, 300), **kw):
    d = dict(n_adapters=4, rank=16, in_=256, n_proj=2, x_dtype=L.ACT_BF16, y_dtype=L.ACT_F32,
             ranks=RANKS, scales=SCALES)
    d.update(kw)
    s = L.Lora(**d)
    for p in range(2):
        s.out[p], s.a[p], s.b[p] = out[p], a[p], b[p]
    return s


def lora(L, x=X, x_ld=256, ids=IDS, T=3, y=(Y0, Y1), y_ld=(100, 300), ws=WS, ws_bytes=1 << 29,
         **kw):
    yp, yl = (C.c_void_p * 4)(*y, None, None), (C.c_int64 * 4)(*y_ld, 0, 0)
    return L.lib().ainfer_moe_lora_apply(C.byref(struct(L, **kw)), x, x_ld, ids, T, yp, yl, ws,
                                         ws_bytes, None)


def test_routing_rows_over_the_bias_or_each_other(L):
    """Workgroups that start late would read what the first ones wrote."""
    row = 4 * 8 * 4
    for kw in (dict(bias=IDX), dict(bias=W), dict(w=IDX), dict(idx=LOGITS), dict(w=LOGITS),
               dict(bias=IDX + row - 4), dict(bias=IDX - 1020), dict(bias=W + row - 4),
               dict(bias=W - 1020), dict(w=IDX + row - 4), dict(w=IDX - row + 4)):
        assert route(L, **kw) == L.ERR_ARG, kw


def test_adapters_written_over_what_is_read(L):
    for out in (Y0, Y1, WS):
        for name in ("x", "ids", "ranks", "scales"):
            assert lora(L, **{name: out}) == L.ERR_ARG, (out, name)
        for p in range(2):
            for name, own in (("a", [A0, A1]), ("b", [B0, B1])):
                own[p] = out
                assert lora(L, **{name: own}) == L.ERR_ARG, (out, name, p)
    assert lora(L, y=(Y0, Y0)) == L.ERR_ARG
    assert lora(L, ws=Y1) == L.ERR_ARG
