"""The operators around the expert stage (scored routing, adapters, the gated
activation) refuse bad arguments before touching the GPU.  CPU only: no call
here reaches a kernel."""
import ctypes as C

import pytest

FAKE = C.c_void_p(0x1000)
ODD = C.c_void_p(0x1001)
TWO = C.c_void_p(0x1002)
EIGHT = C.c_void_p(0x1008)


@pytest.fixture(scope="module")
def L():
    from ainfer_amd import _lib
    return _lib


def routing(L, **kw):
    d = dict(n_experts=256, top_k=8, score=L.SCORE_SIGMOID, n_groups=8, top_groups=4,
             group_score=L.GROUP_TOP2, renormalize=1, scale=2.5)
    d.update(kw)
    return L.Routing(**d)


def route(L, r, logits=FAKE, dtype=0, ld=256, bias=FAKE, T=4, idx=FAKE, w=FAKE):
    return L.lib().ainfer_moe_route_scored(C.byref(r) if r is not None else None, logits, dtype,
                                           ld, bias, T, idx, w, None)


def test_route_scored_refusals(L):
    for bad in (dict(n_experts=0), dict(n_experts=1025), dict(n_experts=1032), dict(n_groups=0),
                dict(n_groups=7), dict(n_groups=65, n_experts=650), dict(n_groups=128),
                dict(top_groups=0), dict(top_groups=9), dict(top_k=0), dict(top_k=33),
                dict(top_k=32, n_experts=64, top_groups=3), dict(top_k=-1), dict(n_groups=-8)):
        assert route(L, routing(L, **bad)) == L.ERR_SHAPE, bad
    for bad in (dict(score=2), dict(score=-1), dict(group_score=2), dict(renormalize=2),
                dict(scale=float("inf")), dict(scale=float("nan"))):
        assert route(L, routing(L, **bad)) == L.ERR_ARG, bad
    r = routing(L)
    assert route(L, None) == L.ERR_NULL
    assert route(L, r, logits=None) == L.ERR_NULL
    assert route(L, r, idx=None) == L.ERR_NULL
    assert route(L, r, w=None) == L.ERR_NULL
    assert route(L, r, T=-1) == L.ERR_TOKENS
    assert route(L, r, T=L.MAX_TOKENS + 1) == L.ERR_TOKENS
    assert route(L, r, T=0, logits=None, idx=None, w=None) == L.OK
    for kw in (dict(dtype=2), dict(dtype=-1), dict(ld=255), dict(ld=-256), dict(ld=1 << 50),
               dict(logits=TWO), dict(logits=ODD, dtype=1), dict(bias=TWO), dict(idx=TWO),
               dict(w=TWO)):
        assert route(L, r, **kw) == L.ERR_ARG, kw


def lora(L, **kw):
    d = dict(n_adapters=4, rank=16, in_=256, n_proj=2, x_dtype=L.ACT_BF16, y_dtype=L.ACT_F32)
    out = kw.pop("out", (100, 300))
    a, b = kw.pop("a", (0x1000, 0x1000)), kw.pop("b", (0x1000, 0x1000))
    d.update(kw)
    s = L.Lora(**d)
    for p in range(2):
        s.out[p], s.a[p], s.b[p] = out[p], a[p], b[p]
    return s


def apply(L, s, x=FAKE, x_ld=256, ids=FAKE, T=3, y=(0x1000, 0x1000), y_ld=(100, 300), ws=FAKE,
          ws_bytes=1 << 40):
    yp = (C.c_void_p * 4)(*y, None, None) if y is not None else None
    yl = (C.c_int64 * 4)(*y_ld, 0, 0) if y_ld is not None else None
    return L.lib().ainfer_moe_lora_apply(C.byref(s) if s is not None else None, x, x_ld, ids, T,
                                         yp, yl, ws, ws_bytes, None)


def test_lora_refusals(L):
    lib = L.lib()
    for bad in (dict(n_adapters=0), dict(n_adapters=4097), dict(rank=0), dict(rank=12),
                dict(rank=136), dict(rank=-8), dict(in_=0), dict(in_=100), dict(in_=65544),
                dict(n_proj=0), dict(n_proj=5), dict(out=(0, 300)), dict(out=(100, (1 << 20) + 1))):
        assert apply(L, lora(L, **bad)) == L.ERR_SHAPE, bad
        assert lib.ainfer_moe_lora_workspace_bytes(C.byref(lora(L, **bad)), 8) == 0, bad
    for bad in (dict(x_dtype=2), dict(y_dtype=-1)):
        assert apply(L, lora(L, **bad)) == L.ERR_ARG, bad
        assert lib.ainfer_moe_lora_workspace_bytes(C.byref(lora(L, **bad)), 8) == 0, bad
    s = lora(L)
    assert apply(L, None) == L.ERR_NULL
    for kw in (dict(x=None), dict(ids=None), dict(y=None), dict(y_ld=None), dict(ws=None),
               dict(y=(0x1000, None))):
        assert apply(L, s, **kw) == L.ERR_NULL, kw
    assert apply(L, lora(L, a=(0x1000, None))) == L.ERR_NULL
    assert apply(L, lora(L, b=(None, 0x1000))) == L.ERR_NULL
    assert apply(L, s, T=-1) == L.ERR_TOKENS
    assert apply(L, s, T=L.MAX_TOKENS + 1) == L.ERR_TOKENS
    assert apply(L, s, T=0, x=None, ids=None, y=None, y_ld=None, ws=None) == L.OK
    for kw in (dict(x=EIGHT), dict(x_ld=255), dict(x_ld=260), dict(x_ld=1 << 50), dict(ids=TWO),
               dict(y=(0x1002, 0x1000)), dict(y_ld=(99, 300)), dict(y_ld=(100, 1 << 50))):
        assert apply(L, s, **kw) == L.ERR_ARG, kw
    assert apply(L, lora(L, a=(0x1008, 0x1000))) == L.ERR_ARG
    assert apply(L, lora(L, b=(0x1000, 0x1004))) == L.ERR_ARG
    assert apply(L, lora(L, ranks=0x1002)) == L.ERR_ARG
    assert apply(L, lora(L, scales=0x1001)) == L.ERR_ARG
    assert apply(L, s, ws=EIGHT) == L.ERR_WORKSPACE
    need = lib.ainfer_moe_lora_workspace_bytes(C.byref(s), 3)
    assert need > 0
    assert apply(L, s, ws_bytes=need - 1) == L.ERR_WORKSPACE
    assert lib.ainfer_moe_lora_workspace_bytes(C.byref(s), -1) == 0
    assert lib.ainfer_moe_lora_workspace_bytes(C.byref(s), L.MAX_TOKENS + 1) == 0
    assert lib.ainfer_moe_lora_workspace_bytes(None, 1) == 0


def test_lora_workspace_grows_with_tokens(L):
    """A workspace for max_tokens serves every call up to it."""
    s = lora(L)
    sizes = [L.lib().ainfer_moe_lora_workspace_bytes(C.byref(s), t)
             for t in (0, 1, 2, 16, 63, 64, 65, 256, 257, 511, 512, 4096, 8191, 8193, 65536)]
    assert sizes == sorted(sizes) and sizes[0] > 0


def silu(L, gate=FAKE, gld=100, up=FAKE, uld=100, dt=0, T=3, I=100, act=FAKE, ald=100, adt=0):
    return L.lib().ainfer_moe_silu_mul(gate, gld, up, uld, dt, T, I, act, ald, adt, None)


def test_silu_mul_refusals(L):
    assert silu(L, T=-1) == L.ERR_TOKENS
    assert silu(L, T=L.MAX_TOKENS + 1) == L.ERR_TOKENS
    assert silu(L, I=0) == L.ERR_SHAPE
    assert silu(L, I=-4) == L.ERR_SHAPE
    for kw in (dict(dt=2), dict(adt=-1), dict(gld=99), dict(uld=99), dict(ald=99),
               dict(gld=1 << 50), dict(gate=TWO), dict(up=TWO), dict(act=TWO),
               dict(act=ODD, adt=1), dict(gate=ODD, dt=1)):
        assert silu(L, **kw) == L.ERR_ARG, kw
    for kw in (dict(gate=None), dict(up=None), dict(act=None)):
        assert silu(L, **kw) == L.ERR_NULL, kw
    assert silu(L, T=0, gate=None, up=None, act=None) == L.OK


def test_python_wrappers_refuse_host_tensors(L):
    torch = pytest.importorskip("torch")
    from ainfer_amd import moe
    x = torch.zeros(2, 8)
    with pytest.raises(L.MoeError):
        moe.silu_mul(x, x, x.clone())
    with pytest.raises(L.MoeError):
        moe.route_scored(L.Routing(8, 2, 0, 1, 1, 0, 1, 1.0), x)
    with pytest.raises(L.MoeError):
        moe.LoraAdapters([torch.zeros(1, 8, 8, dtype=torch.bfloat16)],
                         [torch.zeros(1, 8, 8, dtype=torch.bfloat16)])


def test_overlapping_operands(L):
    """The same address for two operands that a call reads and writes in
    different orders."""
    ys = (0x10000, 0x20000)
    good = dict(x=C.c_void_p(0x40000), ws=C.c_void_p(0x30000))
    for kw in (dict(y=(0x10000, 0x10000)), dict(y=(0x40000, 0x20000)), dict(y=(0x10000, 0x30000)),
               dict(x=C.c_void_p(0x30000))):
        assert apply(L, lora(L), **{**good, "y": ys, **kw}) == L.ERR_ARG, kw
    at = dict(logits=C.c_void_p(0x10000), idx=C.c_void_p(0x20000), w=C.c_void_p(0x30000))
    for kw in (dict(w=at["idx"]), dict(w=at["logits"]), dict(idx=at["logits"])):
        assert route(L, routing(L), **{**at, **kw}) == L.ERR_ARG, kw
    up, act = C.c_void_p(0x10000), FAKE
    for kw in (dict(up=up, act=act, adt=1), dict(up=up, act=act, ald=104),
               dict(gate=up, act=act, adt=1), dict(gate=up, act=act, ald=104)):
        assert silu(L, **kw) == L.ERR_ARG, kw
