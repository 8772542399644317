"""Adapters of more tokens than a batch (ainfer_moe_lora_apply's tiles of 16 tokens),
beside the sizes and values of test_gpu_lora.py."""
import pytest

from test_gpu_lora import Case, torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


# (T, R, K, M): a batch and prompts, in one launch and in two, y in whole pieces of 4
# values and not
@pytest.mark.parametrize("shape", [(256, 8, 64, 100), (257, 8, 64, 100), (700, 24, 136, 99),
                                   (300, 64, 4096, 1028), (300, 64, 4096, 1027),
                                   (513, 56, 72, 65), (600, 128, 1032, 2100)])
@pytest.mark.parametrize("x,y", (("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")))
def test_v_keeps_its_24_bits(torch, shape, x, y):
    """v = 1 + 2^-9 + 2^-18 against -1 - 2^-9 of another rank and of y: every sum is
    exact in fp32, and 2^-18 is left, in either type of y."""
    T, R, K, M = shape
    c = Case(torch, T, 2, R, K, [M], x=x, y=y, ids=[t % 3 - 1 for t in range(T)], scales=False)
    for t in (c.x, c.a[0], c.b[0]):
        t.zero_()
    c.x[:, 0], c.x[:, 3], c.x[:, K - 1] = 1.0, 2.0 ** -9, 2.0 ** -18
    c.a[0][:, 0, [0, 3, K - 1]] = 1.0
    c.a[0][:, R - 1, 0] = 1.0
    c.b[0][:, :, 0] = 1.0
    c.b[0][:, :, R - 1] = -(2.0 ** -9)
    ys = [torch.full_like(c.y[0], -1.0)]
    c.apply(ys)
    torch.cuda.synchronize()
    has = (c.ids >= 0)[:, None].expand_as(ys[0])
    assert (ys[0][has] == 2.0 ** -18).all()
    assert (ys[0][~has] == -1.0).all()


ONE_LAUNCH, TWO_LAUNCHES = (16, 264, [80]), (64, 4096, [1028])  # R, K, rows of y


@pytest.mark.parametrize("T", (33, 257, 300, 700))
@pytest.mark.parametrize("R,K,Ms", (ONE_LAUNCH, (40, 136, [72, 68]), TWO_LAUNCHES))
@pytest.mark.parametrize("y", ("fp32", "bf16"))
def test_rows_inside_wider_ones(torch, T, R, K, Ms, y):
    """x and y of any pitch and y from any column: pieces of 4 values and single ones by
    the rows, the pitch or the address; the columns beside y's stay as they were."""
    for pad, off, x in ((8, 0, "bf16"), (8, 4, "fp32"), (8, 1, "bf16"), (8, 2, "fp32"),
                        (3, 0, "bf16"), (1, 1, "fp32")):
        c = Case(torch, T, 5, R, K, Ms, x=x, y=y, x_pad=8 if pad == 8 else 24)
        wide = [torch.full((T, M + pad + off), 7.0, device="cuda", dtype=c.y[0].dtype) for M in Ms]
        ys = [w[:, off:off + M] for w, M in zip(wide, Ms)]
        for a, b in zip(ys, c.y):
            a.copy_(b)
        c.apply(ys)
        torch.cuda.synchronize()
        c.compare(c.y, [a.contiguous() for a in ys])
        for w, M in zip(wide, Ms):
            assert (w[:, :off] == 7).all() and (w[:, off + M:] == 7).all()


@pytest.mark.parametrize("T", (257, 300, 700))
@pytest.mark.parametrize("R", (8, 16, 24, 32, 48, 64, 72, 128))
def test_ragged_ranks_and_garbage_beyond_them(torch, T, R):
    ranks = [0, 1, 3, R - 1, R, -4, R + 9, R // 2]
    for y in ("fp32", "bf16"):
        c = Case(torch, T, 8, R, 136, [72, 9], ranks=ranks, y=y)
        for n, r in enumerate(ranks):
            r = min(max(r, 0), R)
            for a, b in zip(c.a, c.b):
                a[n, r:] = float("nan")
                b[n, :, r:] = float("inf")
        c.check()


@pytest.mark.parametrize("T", (257, 300, 700))
@pytest.mark.parametrize("R,K,Ms", (ONE_LAUNCH, TWO_LAUNCHES))
@pytest.mark.parametrize("x,y", (("bf16", "fp32"), ("fp32", "bf16"), ("bf16", "bf16")))
def test_other_tokens_of_a_tile_do_not_leak(torch, T, R, K, Ms, x, y):
    """NaN and infinities of one token's x, one adapter's A and another's B beside other
    tokens of the same 16."""
    ids = [t % 7 - 1 for t in range(T)]
    c = Case(torch, T, 6, R, K, Ms, x=x, y=y, ids=ids)
    clean = [v.clone() for v in c.y]
    c.apply(clean)
    bad = {5, 40, T - 2}
    c.x[5], c.x[40, K // 2], c.x[T - 2, 0] = float("nan"), float("inf"), float("-inf")
    c.a[0][1, 0, 3] = float("nan")
    c.b[0][3] = float("inf")
    ys = [v.clone() for v in c.y]
    c.apply(ys)
    torch.cuda.synchronize()
    bad = torch.tensor([ids[t] >= 0 and (t in bad or ids[t] in (1, 3)) for t in range(T)],
                       device="cuda")
    assert torch.equal(ys[0][~bad], clean[0][~bad])
    assert not torch.isfinite(ys[0][bad]).any()


@pytest.mark.parametrize("R,K,M", ((8, 64, 16), (8, 64, 17), (64, 4096, 1028)))
@pytest.mark.parametrize("y", ("fp32", "bf16"))
def test_infinite_and_large_fp32_inputs(torch, R, K, M, y):
    """fp32 x of inf gives inf, the largest finite x what the formula gives, and every bit
    of x counts."""
    T = 300
    c = Case(torch, T, 1, R, K, [M], x="fp32", y=y, ids=[0] * T, ranks=[1], scales=False)
    c.a[0].zero_()
    c.a[0][:, 0, 0] = 1.0
    c.b[0].zero_()
    c.b[0][:, :, 0] = 2.0 ** -10
    c.x.zero_()
    value = [float("inf"), torch.finfo(torch.float32).max, 1 + 2.0 ** -23, -float("inf"),
             1.1754943508222875e-38]
    for t, v in enumerate(value):
        c.x[t, 0] = v
    ys = [torch.zeros_like(c.y[0])]
    c.apply(ys)
    torch.cuda.synchronize()
    want = torch.tensor(value[:4], device="cuda") * 2.0 ** -10
    assert torch.equal(ys[0][:4], want.to(c.y[0].dtype)[:, None].expand(4, M))
    assert (ys[0][4] >= 0).all() and (ys[0][4] <= 2.0 ** -136).all()  # below the normal range
    assert (ys[0][5:] == 0).all()


@pytest.mark.parametrize("T", (257, 400))
@pytest.mark.parametrize("x,y", (("bf16", "fp32"), ("fp32", "bf16")))
def test_every_token_another_adapter(torch, T, x, y):
    """16 adapters to a tile, and neighbours that change places."""
    Case(torch, T, 400, 16, 72, [70], x=x, y=y, ids=list(range(T))).check()
    Case(torch, T, 400, 40, 72, [64], x=x, y=y, ids=[(t * 37) % 400 for t in range(T)]).check()
    Case(torch, T, 2, 16, 72, [64], x=x, y=y, ids=[t % 2 for t in range(T)]).check()


# bytes of 16 rows at a pitch of ld elements of 2 bytes stay below 2^31 up to this one
def last_pitch(n):
    return ((1 << 30) - 1 - n) // 15 // 8 * 8


@pytest.mark.parametrize("which,T,pitch", (("both", 300, (1 << 23) + 8), ("x", 257, "last"),
                                           ("x", 257, "next"), ("y", 257, "last"),
                                           ("y", 257, "next")))
def test_offsets_past_32_bits(torch, which, T, pitch):
    """Rows whose byte offsets pass 2^32, at the last pitch that 16 rows' 32-bit offsets
    reach and at the next one."""
    R, K, M = 8, 64, 48
    c = Case(torch, T, 3, R, K, [M], y="bf16")
    x, ys = c.x, [v.clone() for v in c.y]
    store = []
    for name, n in (("x", K), ("y", M)):
        if which not in (name, "both"):
            continue
        ld = pitch if which == "both" else last_pitch(n) + (8 if pitch == "next" else 0)
        assert which == "both" or ((15 * ld + n) * 2 < (1 << 31) - 1) == (pitch == "last")
        store.append(torch.empty((T - 1) * ld + n, dtype=torch.bfloat16, device="cuda"))
        view = store[-1].as_strided((T, n), (ld, 1))
        if name == "x":
            x = view.copy_(c.x)
        else:
            ys = [view.copy_(c.y[0])]
    c.lora.apply(x, c.ids, ys, c.lora.workspace(T))
    torch.cuda.synchronize()
    c.compare(c.y, [v.contiguous() for v in ys])
    del x, ys, store, view
    torch.cuda.empty_cache()
