"""The 8-bit floating point operators and the token sort refuse bad arguments before
touching the GPU: each operand has an address of its own, and one call differs from a
valid one in one thing.  CPU only: no call here reaches a kernel."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    from ainfer_amd import _lib
    return _lib


def at(n):
    """Operand n of a call: 64 GiB apart, 256-byte aligned."""
    return n << 36


A, B, D, E, F, G, H, W = (at(n) for n in range(1, 9))


def refused(call, cases, status):
    for kw in cases:
        assert call(**kw) == status, kw


def quant(L, x=A, x_ld=512, dtype=0, live=B, N=4, K=512, kind=0, q=D, q_ld=512, sq=E):
    return L.lib().ainfer_moe_act_quant_fp8(x, x_ld, dtype, live, N, K, kind, q, q_ld, sq, None)


def test_act_quant(L):
    call = lambda **kw: quant(L, **kw)  # noqa: E731
    refused(call, (dict(N=-1), dict(N=L.MAX_ROWS + 1)), L.ERR_TOKENS)
    refused(call, (dict(K=0), dict(K=8), dict(K=504), dict(K=65552), dict(K=-16)), L.ERR_SHAPE)
    refused(call, (dict(x=None), dict(q=None), dict(sq=None)), L.ERR_NULL)
    refused(call, (dict(dtype=2), dict(dtype=-1), dict(kind=2), dict(kind=-1), dict(x_ld=511),
                   dict(x_ld=-512), dict(x_ld=1 << 40), dict(q_ld=511), dict(q_ld=520),
                   dict(q_ld=1 << 40), dict(x=A + 2), dict(x=A + 1, dtype=1), dict(q=D + 8),
                   dict(sq=E + 2), dict(live=B + 2), dict(q=A), dict(sq=A), dict(sq=D + 2032),
                   dict(sq=A + 8188), dict(live=E + 60), dict(live=D + 4), dict(q=A + 512),
                   dict(x=D + 1024), dict(q=A + 8176, q_ld=512)), L.ERR_ARG)
    assert quant(L, N=0, x=None, q=None, sq=None) == L.OK


def silu(L, g=A, g_ld=512, u=B, u_ld=512, dtype=0, live=G, N=4, I=512, kind=0, q=D, q_ld=512, sq=E):
    return L.lib().ainfer_moe_silu_mul_fp8(g, g_ld, u, u_ld, dtype, live, N, I, kind, q, q_ld, sq,
                                           None)


def test_silu_mul_fp8(L):
    call = lambda **kw: silu(L, **kw)  # noqa: E731
    refused(call, (dict(N=-1), dict(N=L.MAX_ROWS + 1)), L.ERR_TOKENS)
    refused(call, (dict(I=0), dict(I=100), dict(I=65552)), L.ERR_SHAPE)
    refused(call, (dict(g=None), dict(u=None), dict(q=None), dict(sq=None)), L.ERR_NULL)
    refused(call, (dict(dtype=2), dict(kind=3), dict(g_ld=511), dict(u_ld=511), dict(q_ld=500),
                   dict(q_ld=520), dict(g=A + 2), dict(u=B + 1), dict(q=D + 4), dict(sq=E + 1),
                   dict(live=G + 1), dict(q=A), dict(q=B), dict(sq=A), dict(sq=B), dict(live=E),
                   dict(live=D), dict(sq=D + 16), dict(q=A + 16), dict(u=D - 16)), L.ERR_ARG)
    assert silu(L, N=0, g=None, u=None, q=None, sq=None) == L.OK


def grad(L, d=A, d_ld=64, g=B, g_ld=64, u=D, u_ld=64, dtype=0, live=G, N=4, I=64, dg=E, dg_ld=64,
         du=F, du_ld=64):
    return L.lib().ainfer_moe_silu_mul_backward(d, d_ld, g, g_ld, u, u_ld, dtype, live, N, I, dg,
                                                dg_ld, du, du_ld, None)


def test_silu_mul_backward(L):
    call = lambda **kw: grad(L, **kw)  # noqa: E731
    refused(call, (dict(N=-1), dict(N=L.MAX_ROWS + 1)), L.ERR_TOKENS)
    refused(call, (dict(I=0), dict(I=-1), dict(I=65537)), L.ERR_SHAPE)
    refused(call, (dict(d=None), dict(g=None), dict(u=None), dict(dg=None), dict(du=None)),
            L.ERR_NULL)
    refused(call, (dict(dtype=2), dict(d_ld=63), dict(g_ld=63), dict(u_ld=63), dict(dg_ld=63),
                   dict(du_ld=63), dict(d=A + 1), dict(g=B + 2), dict(u=D + 3), dict(dg=E + 1),
                   dict(du=F + 2), dict(live=G + 2), dict(du=E), dict(dg=A, dg_ld=65),
                   dict(du=D, du_ld=70), dict(dg=B, g_ld=66), dict(live=E + 8), dict(live=F)),
            L.ERR_ARG)
    assert grad(L, N=0, d=None, g=None, u=None, dg=None, du=None) == L.OK


def weights(L, w=A, dtype=0, E_=2, M=130, K=272, kind=0, q=B, s=D):
    return L.lib().ainfer_moe_weight_quant_fp8(w, dtype, E_, M, K, kind, q, s, None)


SIZES = (dict(E_=0), dict(E_=1025), dict(M=0), dict(M=(1 << 20) + 1), dict(K=0), dict(K=20),
         dict(K=65552), dict(E_=1024, M=1 << 20, K=65536))


def test_weight_quant(L):
    call = lambda **kw: weights(L, **kw)  # noqa: E731
    refused(call, SIZES, L.ERR_SHAPE)
    refused(call, (dict(w=None), dict(q=None), dict(s=None)), L.ERR_NULL)
    refused(call, (dict(dtype=2), dict(kind=2), dict(w=A + 2), dict(q=B + 8), dict(s=D + 2),
                   dict(q=A), dict(q=A + 16), dict(s=A), dict(s=B + 64)), L.ERR_ARG)


def pack(L, w=A, E_=2, M=130, K=272, t=0, p=B, n=1 << 30):
    return L.lib().ainfer_moe_fp8_pack(w, E_, M, K, t, p, n, None)


def test_pack(L):
    call = lambda **kw: pack(L, **kw)  # noqa: E731
    refused(call, SIZES, L.ERR_SHAPE)
    refused(call, (dict(w=None), dict(p=None)), L.ERR_NULL)
    n = L.lib().ainfer_moe_fp8_packed_bytes(2, 130, 272)
    assert n == 2 * 192 * 384
    refused(call, (dict(t=2), dict(t=-1), dict(w=A + 8), dict(p=B + 8), dict(n=n - 1), dict(p=A),
                   dict(p=A + 65536), dict(w=B + 16)), L.ERR_ARG)
    for kw in SIZES:
        d = dict(E_=2, M=130, K=272)
        d.update(kw)
        assert L.lib().ainfer_moe_fp8_packed_bytes(d["E_"], d["M"], d["K"]) == 0


def product(L, E_=2, M=130, K=272, dtype=1, w=A, s=B, q=D, q_ld=272, sq=E, offsets=F, N=5, y=G,
            y_ld=130, struct=True):
    d = L.Fp8(E_, M, K, dtype, w, s)
    return L.lib().ainfer_moe_fp8_product(C.byref(d) if struct else None, q, q_ld, sq, offsets, N, y,
                                          y_ld, None)


def test_product(L):
    call = lambda **kw: product(L, **kw)  # noqa: E731
    refused(call, SIZES, L.ERR_SHAPE)
    refused(call, (dict(N=-1), dict(N=L.MAX_ROWS + 1)), L.ERR_TOKENS)
    refused(call, (dict(struct=False), dict(w=None), dict(s=None), dict(q=None), dict(sq=None),
                   dict(offsets=None), dict(y=None)), L.ERR_NULL)
    refused(call, (dict(dtype=2), dict(dtype=-1), dict(q_ld=256), dict(q_ld=280), dict(q_ld=(1 << 24) + 16),
                   dict(y_ld=129), dict(y_ld=1 << 40), dict(y=D + 16), dict(q=G + 1280), dict(w=A + 8), dict(q=D + 8), dict(s=B + 2), dict(sq=E + 2),
                   dict(offsets=F + 2), dict(y=G + 1), dict(y=D), dict(y=A), dict(y=A + 256),
                   dict(y=B), dict(y=E), dict(y=F), dict(y=F - 1024), dict(y=A, y_ld=140),
                   dict(y=F, y_ld=140)), L.ERR_ARG)
    assert product(L, N=0, w=None, s=None, q=None, sq=None, offsets=None, y=None) == L.OK
    assert product(L, N=0, dtype=3) == L.ERR_ARG


def sort(L, E_=64, k=4, H_=272, dtype=1, fp8=1, kind=0, x=A, x_ld=272, idx=B, T=8, off=D, pos=E,
         rows=F, r_ld=272, sc=G, ws=W, ws_bytes=1 << 20, struct=True):
    d = L.Sorting(E_, k, H_, dtype, fp8, kind)
    return L.lib().ainfer_moe_sort_rows(C.byref(d) if struct else None, x, x_ld, idx, T, off, pos,
                                        rows, r_ld, sc, ws, ws_bytes, None)


def test_sort_rows(L):
    call = lambda **kw: sort(L, **kw)  # noqa: E731
    refused(call, (dict(E_=0), dict(E_=1025), dict(k=0), dict(k=33), dict(H_=0), dict(H_=65552),
                   dict(H_=264)), L.ERR_SHAPE)
    refused(call, (dict(T=-1), dict(T=L.MAX_TOKENS + 1)), L.ERR_TOKENS)
    refused(call, (dict(struct=False), dict(x=None), dict(idx=None), dict(off=None),
                   dict(pos=None), dict(sc=None), dict(ws=None)), L.ERR_NULL)
    refused(call, (dict(dtype=2), dict(fp8=2), dict(kind=2), dict(x_ld=271), dict(r_ld=271),
                   dict(r_ld=280), dict(x=A + 1), dict(rows=F + 8), dict(sc=G + 2),
                   dict(idx=B + 2), dict(off=D + 1), dict(pos=E + 2), dict(x_ld=1 << 40)),
            L.ERR_ARG)
    refused(call, (dict(ws=W + 16), dict(ws_bytes=1)), L.ERR_WORKSPACE)
    # what is written over another operand
    refused(call, (dict(off=E), dict(off=B), dict(pos=B), dict(pos=D + 256), dict(ws=D),
                   dict(ws=E), dict(ws=B), dict(sc=D), dict(sc=E), dict(sc=B), dict(sc=W),
                   dict(rows=A), dict(rows=A + 16), dict(rows=D), dict(rows=E), dict(rows=W),
                   dict(rows=G), dict(rows=B), dict(rows=B, r_ld=288), dict(off=A), dict(pos=A),
                   dict(ws=A), dict(sc=A), dict(sc=F + 16), dict(pos=F + 32)), L.ERR_ARG)
    assert L.lib().ainfer_moe_sort_workspace_bytes(8, 4, 64) > 0
    for bad in ((-1, 4, 64), (L.MAX_TOKENS + 1, 4, 64), (8, 0, 64), (8, 33, 64), (8, 4, 0),
                (8, 4, 1025)):
        assert L.lib().ainfer_moe_sort_workspace_bytes(*bad) == 0, bad


def back(L, rows=A, r_ld=64, rdt=1, N=40, pos=B, w=D, T=10, k=4, H_=64, resid=E, s_ld=64, y=F,
         y_ld=64, ydt=0):
    return L.lib().ainfer_moe_unpermute(rows, r_ld, rdt, N, pos, w, T, k, H_, resid, s_ld, y, y_ld,
                                        ydt, None)


def test_unpermute(L):
    call = lambda **kw: back(L, **kw)  # noqa: E731
    refused(call, (dict(T=-1), dict(T=L.MAX_TOKENS + 1), dict(N=-1), dict(N=L.MAX_ROWS + 1)),
            L.ERR_TOKENS)
    refused(call, (dict(k=0), dict(k=33), dict(H_=0), dict(H_=65537)), L.ERR_SHAPE)
    refused(call, (dict(rows=None), dict(pos=None), dict(y=None)), L.ERR_NULL)
    refused(call, (dict(rdt=2), dict(ydt=-1), dict(r_ld=63), dict(s_ld=63), dict(y_ld=63),
                   dict(rows=A + 1), dict(pos=B + 2), dict(w=D + 2), dict(resid=E + 2),
                   dict(y=F + 2), dict(y=A), dict(y=A + 64), dict(y=B), dict(y=D + 8),
                   dict(resid=F, s_ld=65), dict(y=B, y_ld=70)), L.ERR_ARG)
    assert back(L, T=0, rows=None, pos=None, y=None) == L.OK


def back_grad(L, dy=A, y_ld=64, ydt=0, rows=B, r_ld=64, rdt=1, N=40, pos=D, w=E, T=10, k=4, H_=64,
              dr=F, d_ld=64, dw=G):
    return L.lib().ainfer_moe_unpermute_backward(dy, y_ld, ydt, rows, r_ld, rdt, N, pos, w, T, k,
                                                 H_, dr, d_ld, dw, None)


def test_unpermute_backward(L):
    call = lambda **kw: back_grad(L, **kw)  # noqa: E731
    refused(call, (dict(T=-1), dict(T=L.MAX_TOKENS + 1), dict(N=-1), dict(N=L.MAX_ROWS + 1)),
            L.ERR_TOKENS)
    refused(call, (dict(k=0), dict(k=33), dict(H_=0), dict(H_=65537)), L.ERR_SHAPE)
    refused(call, (dict(dy=None), dict(pos=None), dict(rows=None)), L.ERR_NULL)
    refused(call, (dict(rdt=2), dict(ydt=2), dict(r_ld=63), dict(y_ld=63), dict(d_ld=63),
                   dict(dy=A + 2), dict(rows=B + 1), dict(dr=F + 1), dict(pos=D + 1),
                   dict(w=E + 2), dict(dw=G + 2), dict(dw=D), dict(dw=E + 4), dict(dw=A),
                   dict(dw=B + 128), dict(dr=A), dict(dr=A + 64), dict(dr=B), dict(dr=B + 2),
                   dict(dr=D), dict(dr=E), dict(dr=G)), L.ERR_ARG)
    assert back_grad(L, T=0, dy=None, pos=None, rows=None) == L.OK
    assert back_grad(L, dr=None, dw=None) == L.OK


def test_host_tensors_and_wrong_types():
    """The Python surface refuses tensors that the kernels could not read."""
    import torch
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    x, i = torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int32)
    w = torch.zeros(1, 64, 64, dtype=torch.uint8)
    b = torch.zeros(256, dtype=torch.uint8)
    for call in (lambda: moe.act_quant_fp8(x), lambda: moe.silu_mul_fp8(x, x),
                 lambda: moe.silu_mul_backward(x, x, x, x, x),
                 lambda: moe.weight_quant_fp8(x[None]),
                 lambda: moe.Fp8Weights(w, torch.zeros(1, 1, 1)),
                 lambda: moe.sort_rows(x, i, 8, b), lambda: moe.unpermute(x, i, None, x),
                 lambda: moe.unpermute_backward(x, x, i, None, x),
                 lambda: moe.sort_workspace(4, 2, 0), lambda: moe.sort_workspace(-1, 2, 8)):
        with pytest.raises(L.MoeError):
            call()
