"""Calls that reach each form of the 8-bit product, small enough for a test."""
import ctypes as C


def form(E, M, K, N, dtype):
    """(weight rows, rows) of the form's items; dtype: "float32" or "bfloat16"."""
    from ainfer_amd import _lib as L
    m, rows = C.c_int32(), C.c_int32()
    L.check(L.lib().ainfer_moe_debug_fp8_form(
        E, M, K, N, L.ACT_F32 if dtype == "float32" else L.ACT_BF16, C.byref(m), C.byref(rows)))
    return m.value, rows.value


TWO = [400, 300]  # rows of two experts

# (y's type, form, rows of each expert, M); K is the test's: 272 here, three groups, one of 16 columns
CALLS = (
    ("bfloat16", (256, 128), TWO, 9000),
    ("bfloat16", (256, 96), TWO, 4100),
    ("bfloat16", (64, 32), TWO, 1000),
    ("bfloat16", (32, 32), TWO, 512),
    ("bfloat16", (32, 16), TWO, 300),
    ("bfloat16", (16, 16), [9], 300),
    ("float32", (256, 96), TWO, 19200),
    ("float32", (256, 64), TWO, 9000),
    ("float32", (64, 32), TWO, 1000),
    ("float32", (32, 32), TWO, 512),
    ("float32", (32, 16), TWO, 300),
    ("float32", (16, 16), [9], 300),
)

# one busy expert among hundreds without rows
BUSY = (
    ("bfloat16", (256, 128), [0] * 200 + [6900] + [0] * 199, 1030),
    ("bfloat16", (256, 96), [0] * 399 + [5400], 1030),
    ("float32", (256, 96), [0] * 77 + [26100] + [0] * 322, 300),
    ("float32", (256, 64), [6900] + [0] * 399, 1030),
    ("bfloat16", (64, 32), [0, 0, 700, 0], 800),
    ("bfloat16", (32, 16), [0] * 500 + [3000] + [0] * 523, 70),
    ("float32", (32, 16), [0] * 500 + [3000] + [0] * 523, 70),
)


def name(call):
    dtype, (m, rows), counts, M = call
    return f"{dtype}-{m}x{rows}-{len(counts)}e{sum(counts)}-{M}"


def reached(call, K, extra=0):
    """Fails where the rule sends the call elsewhere."""
    dtype, want, counts, M = call
    assert form(len(counts), M, K, sum(counts) + extra, dtype) == want, call
