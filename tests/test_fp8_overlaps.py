"""Rows that are written over rows that are read, or over each other, are refused wherever they meet,
not at equal addresses alone.  CPU only: no call here reaches a kernel."""
import pytest

import test_fp8_refusals as R
from test_fp8_refusals import A, B, D, E, F, G, L  # noqa: F401  (L: the fixture)

# 4 rows of 64 fp32 values: 1024 bytes where they are whole
WHOLE = 4 * 64 * 4


@pytest.mark.parametrize("out,ld", (("dg", "dg_ld"), ("du", "du_ld")))
def test_silu_mul_backward(L, out, ld):  # noqa: F811
    for at in (A, B, D):  # dact, gate, up
        R.refused(lambda **kw: R.grad(L, **kw), (
            {out: at + 4}, {out: at - 4}, {out: at + 64}, {out: at + WHOLE - 4},
            {out: at - WHOLE + 4},
            # rows with room between them, the last one behind the first input row's start
            {out: at - 3 * 400, ld: 100}, {out: at + 1000, ld: 100}), L.ERR_ARG)
    # rows of one pitch: an input's columns 1.. and columns behind its row
    for d in (4, 252, -252, 600, 400 - 4, 3 * 400 + 252, -3 * 400 - 252):
        R.refused(lambda **kw: R.grad(L, **kw), (
            {out: A + d, ld: 100, "d_ld": 100}, {out: B + d, ld: 100, "g_ld": 100},
            {out: D + d, ld: 100, "u_ld": 100}), L.ERR_ARG)


def test_silu_mul_backward_outputs(L):  # noqa: F811
    """The two gradients over each other."""
    R.refused(lambda **kw: R.grad(L, **kw), (
        dict(dg=E, du=E), dict(dg=E, du=E + 64), dict(dg=E + 64, du=E), dict(dg=B + 64, du=B + 128),
        dict(dg=E, du=E + 128, dg_ld=100, du_ld=100), dict(dg=E, du=E + 3 * 400 + 252, dg_ld=100, du_ld=100),
        dict(dg=E, du=E + 900, dg_ld=100), dict(dg=E + 900, du=E, du_ld=100),
        dict(dg=E, du=E, N=1), dict(dg=E, du=E + 252, N=1)), L.ERR_ARG)


def test_unpermute(L):  # noqa: F811
    # 10 rows of 64 fp32 values at y, 40 rows of 64 bf16 values at rows
    R.refused(lambda **kw: R.back(L, **kw), (
        dict(resid=F + 4), dict(resid=F - 4), dict(resid=F + 2556), dict(y=E + 64), dict(y=E - 64),
        dict(resid=F + 4, s_ld=100, y_ld=100), dict(resid=F + 252, s_ld=100, y_ld=100),
        dict(resid=F + 9 * 400, s_ld=100, y_ld=100), dict(resid=F - 9 * 400 - 252, s_ld=100, y_ld=100),
        dict(resid=F - 900, s_ld=100), dict(resid=F + 900, y_ld=100),
        dict(resid=F + 4, T=1), dict(resid=F - 252, T=1)), L.ERR_ARG)
    R.refused(lambda **kw: R.back(L, **kw), (
        dict(y=A + 64, r_ld=200, y_ld=100), dict(y=A + 39 * 400 + 124, r_ld=200, y_ld=100),
        dict(y=B + 156, y_ld=100), dict(y=B - 9 * 400 - 252, y_ld=100), dict(y=D + 100, y_ld=100)),
        L.ERR_ARG)


def test_pitched_rows_of_the_other_calls(L):  # noqa: F811
    """Past the first row's address too, where rows have room between them."""
    # 4 rows of 512 codes, 512 fp32 values
    R.refused(lambda **kw: R.quant(L, **kw), (
        dict(q=A + 2032, x_ld=1024, q_ld=4096), dict(q=A + 12288 + 2032, x_ld=1024, q_ld=4096),
        dict(sq=D + 3 * 1024, q_ld=1024), dict(live=D + 3 * 1024 + 508, q_ld=1024),
        dict(q=E - 3 * 1024, q_ld=1024), dict(sq=A + 4096 + 2044, x_ld=1024)), L.ERR_ARG)
    R.refused(lambda **kw: R.silu(L, **kw), (
        dict(q=B + 4096, u_ld=1024, q_ld=4096), dict(sq=D + 1024, q_ld=1024),
        dict(sq=A + 4096, g_ld=1024), dict(live=D + 2048, q_ld=1024)), L.ERR_ARG)
    # 5 rows of 130 bf16 values at y, of 272 codes at q
    R.refused(lambda **kw: R.product(L, **kw), (
        dict(y=D + 512, q_ld=512, y_ld=256), dict(y=D + 4 * 512 + 270, q_ld=512, y_ld=256),
        dict(y=F - 2048, y_ld=256), dict(y=E - 512 - 258, y_ld=256)), L.ERR_ARG)
    # 32 rows of 272 codes, 8 rows of 272 bf16 values
    R.refused(lambda **kw: R.sort(L, **kw), (
        dict(rows=A + 512 * 3, x_ld=512, r_ld=1024), dict(rows=E - 1024, r_ld=1024),
        dict(off=A + 2048, x_ld=512), dict(rows=G - 31 * 1024, r_ld=1024)), L.ERR_ARG)
    # 40 rows of 64 bf16 values, 10 rows of 64 fp32 values
    R.refused(lambda **kw: R.back_grad(L, **kw), (
        dict(dr=A + 400, d_ld=200, y_ld=100), dict(dr=B + 126, d_ld=200, r_ld=200),
        dict(dr=G - 39 * 400 - 126, d_ld=200), dict(dw=B + 39 * 400, r_ld=200), dict(dr=E - 400, d_ld=200),
        dict(dr=D - 126 - 400, d_ld=200)), L.ERR_ARG)
