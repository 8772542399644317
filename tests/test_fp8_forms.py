"""The rule between the forms of the 8-bit product: the calls of the tests of each form reach it,
and the sizes that it names take the form that was faster there.  CPU only."""
import ctypes as C

import pytest

import fp8_forms as F


@pytest.mark.parametrize("call", F.CALLS + F.BUSY, ids=F.name)
def test_calls_reach_their_form(call):
    F.reached(call, 272, extra=5)


def test_every_form_is_tested():
    for dtype, tiles in (("bfloat16", {(256, 128), (256, 96)}), ("float32", {(256, 96), (256, 64)})):
        want = tiles | {(64, 32), (32, 32), (32, 16), (16, 16)}
        assert {c[1] for c in F.CALLS if c[0] == dtype} == want


# (experts, K, M, rows, form) at the sizes that the rule's comment gives times for
NAMED = {"bfloat16": ((1, 4096, 4096, 256, (64, 32)), (1, 4096, 4096, 512, (256, 96)), (1, 5120, 17408, 64, (256, 96)),
                      (16, 2048, 2048, 288, (256, 96)), (64, 4096, 2048, 2048, (256, 128)),
                      (256, 2048, 1024, 128, (32, 16)), (512, 2048, 1024, 512, (32, 16)),
                      (64, 4096, 2048, 512, (32, 16)), (1, 4096, 4096, 2048, (256, 128)),
                      (64, 4096, 2048, 8192, (256, 128)), (1, 4096, 4096, 1024, (256, 96)),
                      (512, 2048, 1024, 4096, (256, 96)), (1, 5120, 17408, 1, (16, 16)),
                      (1, 4096, 4096, 32, (32, 16)), (1, 4096, 4096, 64, (32, 32)),
                      (1, 4096, 4096, 128, (64, 32))),
         "float32": ((4, 4096, 4096, 256, (64, 32)), (16, 2048, 2048, 288, (256, 64)),
                     (64, 4096, 2048, 16384, (256, 96)), (64, 4096, 2048, 8192, (256, 96)),
                     (1, 4096, 4096, 8192, (256, 96)), (1, 4096, 4096, 2048, (256, 64)),
                     (96, 2560, 1792, 5952, (256, 64)))}


@pytest.mark.parametrize("dtype", NAMED)
def test_named_sizes(dtype):
    for E, K, M, N, want in NAMED[dtype]:
        assert F.form(E, M, K, N, dtype) == want, (E, K, M, N)


def test_refusals():
    from ainfer_amd import _lib as L
    a, b = C.c_int32(), C.c_int32()

    def call(E=1, M=64, K=128, N=5, dt=0, p=C.byref(a), q=C.byref(b)):
        return L.lib().ainfer_moe_debug_fp8_form(E, M, K, N, dt, p, q)

    assert call() == L.OK
    for kw in (dict(E=0), dict(M=0), dict(K=20), dict(K=65552)):
        assert call(**kw) == L.ERR_SHAPE
    assert call(N=0) == call(N=L.MAX_ROWS + 1) == L.ERR_TOKENS
    assert call(dt=2) == L.ERR_ARG and call(p=None) == call(q=None) == L.ERR_NULL
