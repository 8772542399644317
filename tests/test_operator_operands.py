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


@pytest.fixture
def no_gpu():
    """A call that passes every check gets as far as a launch only here."""
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU would run the call on addresses that hold nothing")


def test_valid_calls_pass_every_check(L, no_gpu):
    """They end at the launch, which needs a GPU."""
    for kw in (dict(), dict(dtype=1), dict(bias=None), dict(ld=1 << 40), dict(T=L.MAX_TOKENS),
               dict(score=L.SCORE_SOFTMAX, group_score=L.GROUP_MAX, renormalize=0),
               dict(dtype=1, logits=LOGITS + 2, bias=BIAS + 4, idx=IDX + 4, w=W + 4),
               dict(n_experts=1024, n_groups=64, top_groups=2, top_k=32, ld=1024),
               dict(n_experts=1, n_groups=1, top_groups=1, top_k=1, ld=1)):
        assert route(L, **kw) == L.ERR_HIP, kw
    for kw in (dict(), dict(ranks=None, scales=None), dict(x_ld=264), dict(x_ld=260, x_dtype=0),
               dict(y=(Y0 + 4, Y1 + 4)), dict(y=(Y0 + 2, Y1 + 2), y_dtype=1), dict(T=L.MAX_TOKENS),
               dict(n_adapters=4096, rank=128, in_=65536, x_ld=65536)):
        assert lora(L, **kw) == L.ERR_HIP, kw
    for kw in (dict(), dict(up=GATE), dict(act=GATE), dict(act=UP, adt=0), dict(adt=1),
               dict(act=GATE, adt=1, dt=1), dict(gate=GATE + 2, up=UP + 2, act=ACT + 2, dt=1, adt=1),
               dict(gld=101, uld=104, ald=1 << 40), dict(act=GATE, T=1, ald=104)):
        assert silu(L, **kw) == L.ERR_HIP, kw


def test_route_scored_refuses_each_argument(L):
    for kw in (dict(n_experts=0), dict(n_experts=-8), dict(n_experts=1032, ld=1032), dict(n_groups=0),
               dict(n_groups=-8), dict(n_groups=7), dict(n_groups=128, top_groups=64),
               dict(top_groups=0), dict(top_groups=9), dict(top_k=0), dict(top_k=-1),
               dict(top_k=33), dict(top_k=32, n_experts=64, top_groups=3)):
        assert route(L, **kw) == L.ERR_SHAPE, kw
    for kw in (dict(T=-1), dict(T=L.MAX_TOKENS + 1)):
        assert route(L, **kw) == L.ERR_TOKENS, kw
    for kw in (dict(score=2), dict(score=-1), dict(group_score=2), dict(group_score=-1),
               dict(renormalize=2), dict(renormalize=-1), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(dtype=2), dict(dtype=-1), dict(ld=255), dict(ld=0),
               dict(ld=-256), dict(ld=(1 << 40) + 1), dict(logits=LOGITS + 2),
               dict(logits=LOGITS + 1, dtype=1), dict(bias=BIAS + 2), dict(idx=IDX + 2),
               dict(w=W + 2)):
        assert route(L, **kw) == L.ERR_ARG, kw
    for kw in (dict(logits=None), dict(idx=None), dict(w=None)):
        assert route(L, **kw) == L.ERR_NULL, kw
    assert route(L, T=0, logits=None, idx=None, w=None) == L.OK
    assert L.lib().ainfer_moe_route_scored(None, LOGITS, 0, 256, BIAS, 4, IDX, W,
                                           None) == L.ERR_NULL


def test_lora_refuses_each_argument(L):
    lib = L.lib()
    need = lib.ainfer_moe_lora_workspace_bytes(C.byref(struct(L)), 3)
    assert need == lib.ainfer_moe_lora_workspace_bytes(C.byref(struct(L, ranks=None)), 3) > 0
    # every other check passes, and the workspace's comes after them
    for kw in (dict(ws_bytes=need - 1), dict(ws_bytes=0), dict(ws=WS + 8), dict(ws=WS + 128)):
        assert lora(L, **kw) == L.ERR_WORKSPACE, kw
    for kw in (dict(n_adapters=0), dict(n_adapters=4097), dict(rank=0), dict(rank=-8),
               dict(rank=12), dict(rank=136), dict(in_=0), dict(in_=100), dict(in_=65544, x_ld=65544),
               dict(n_proj=0), dict(n_proj=5), dict(out=(0, 300)), dict(out=(100, -1)),
               dict(out=(100, (1 << 20) + 1), y_ld=(100, 1 << 21))):
        assert lora(L, **kw) == L.ERR_SHAPE, kw
    for kw in (dict(T=-1), dict(T=L.MAX_TOKENS + 1)):
        assert lora(L, **kw) == L.ERR_TOKENS, kw
    for kw in (dict(x_dtype=2), dict(x_dtype=-1), dict(y_dtype=2), dict(y_dtype=-1),
               dict(x=X + 8), dict(x_ld=248), dict(x_ld=260), dict(x_ld=(1 << 40) + 8),
               dict(ids=IDS + 2), dict(ranks=RANKS + 2), dict(scales=SCALES + 1),
               dict(a=(A0 + 8, A1)), dict(a=(A0, A1 + 2)), dict(b=(B0 + 8, B1)),
               dict(b=(B0, B1 + 4)), dict(y=(Y0 + 2, Y1)), dict(y=(Y0, Y1 + 1), y_dtype=1),
               dict(y_ld=(99, 300)), dict(y_ld=(100, 299)), dict(y_ld=(100, (1 << 40) + 1))):
        # also with a workspace that would be refused later
        assert lora(L, **kw) == L.ERR_ARG, kw
        assert lora(L, ws_bytes=need - 1, **kw) == L.ERR_ARG, kw
    for kw in (dict(x=None), dict(ids=None), dict(ws=None), dict(y=(None, Y1)), dict(y=(Y0, None)),
               dict(a=(None, A1)), dict(a=(A0, None)), dict(b=(None, B1)), dict(b=(B0, None))):
        assert lora(L, **kw) == L.ERR_NULL, kw
    assert lora(L, T=0, x=None, ids=None, y=(None, None), ws=None) == L.OK
    s, yp, yl = struct(L), (C.c_void_p * 4)(Y0, Y1), (C.c_int64 * 4)(100, 300)
    assert lib.ainfer_moe_lora_apply(None, X, 256, IDS, 3, yp, yl, WS, 1 << 29, None) == L.ERR_NULL
    for y, ld in ((None, yl), (yp, None)):
        assert lib.ainfer_moe_lora_apply(C.byref(s), X, 256, IDS, 3, y, ld, WS, 1 << 29,
                                         None) == L.ERR_NULL
    for n in (-1, L.MAX_TOKENS + 1):
        assert lib.ainfer_moe_lora_workspace_bytes(C.byref(s), n) == 0
    for bad in (dict(rank=12), dict(n_adapters=0), dict(x_dtype=2)):
        assert lib.ainfer_moe_lora_workspace_bytes(C.byref(struct(L, **bad)), 3) == 0, bad


GATE, UP, ACT = (at(n) for n in range(31, 34))


def silu(L, gate=GATE, gld=100, up=UP, uld=100, dt=0, T=3, I=100, act=ACT, ald=100, adt=0):
    return L.lib().ainfer_moe_silu_mul(gate, gld, up, uld, dt, T, I, act, ald, adt, None)


def test_silu_mul_refuses_each_argument(L):
    for kw in (dict(T=-1), dict(T=L.MAX_TOKENS + 1)):
        assert silu(L, **kw) == L.ERR_TOKENS, kw
    for kw in (dict(I=0), dict(I=-4)):
        assert silu(L, **kw) == L.ERR_SHAPE, kw
    big = (1 << 40) + 1
    for kw in (dict(dt=2), dict(dt=-1), dict(adt=2), dict(adt=-1), dict(gld=99), dict(uld=99),
               dict(ald=99), dict(gld=big), dict(uld=big), dict(ald=big), dict(gate=GATE + 2),
               dict(up=UP + 2), dict(act=ACT + 2), dict(gate=GATE + 1, dt=1),
               dict(up=UP + 1, dt=1), dict(act=ACT + 1, adt=1),
               # in place with elements of another size or rows at other places
               dict(act=GATE, adt=1), dict(act=UP, adt=1), dict(act=GATE, dt=1),
               dict(act=UP, dt=1), dict(act=GATE, ald=104), dict(act=UP, ald=104),
               dict(act=GATE, gld=104), dict(act=UP, uld=104)):
        assert silu(L, **kw) == L.ERR_ARG, kw
    for kw in (dict(gate=None), dict(up=None), dict(act=None)):
        assert silu(L, **kw) == L.ERR_NULL, kw
    assert silu(L, T=0, gate=None, up=None, act=None) == L.OK
