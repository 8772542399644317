"""8-bit floating point rows, weights and products against their definitions.

Bounds.  Codes and scales of given rows: the definition's own bits.  Codes of a
gated activation: its fp32 value is off by 2^-21 (test_gpu_silu.py), so a code may be
the neighbour at a tie: 2^-4 of the value by the code's rounding (half a step; 2^-10
scales near zero), and what that value is off.  Products: 128 additions of a group in
fp32, the product of the scales, and one fma a group, each off by 2^-24 of the sum of
magnitudes at most: (128 + G + 4) 2^-24 of it.  bf16 outputs come from an instruction that
drops what is more than 13 bits below the largest of eight products: seven others lose
less than 2^-13 of the largest each, 7 * 2^-13 of the sum of magnitudes at most, and
one rounding more, 2^-8.  That is wide enough to hide a column in a thousand, so their
norm is bounded too: the dropped parts' signs are the products', which are random here, so
their squares add up: sqrt(7) 2^-13 of the largest product in each eight, less than
2^-11 of the norm of the result, whose square is at least those largest products' squares
together."""
import pytest

import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def same_codes(torch, got, want):
    got, want = got.cpu().float(), want.float()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    # minus zero too
    assert torch.equal(torch.signbit(got.nan_to_num()), torch.signbit(want.nan_to_num()))


@pytest.mark.parametrize("pow2", (False, True))
@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("n,K", ((1, 16), (1, 128), (3, 144), (5, 4096), (17, 2000), (300, 272),
                                 (1, 65536), (2049, 128)))
def test_act_quant(torch, n, K, dtype, pow2):
    from ainfer_amd import moe
    print(f"[case] quant {n} x {K} {dtype} pow2 {pow2}", flush=True)
    x = torch.randn(n, K, generator=gen(torch, n + K), device="cuda").to(getattr(torch, dtype))
    q, s = moe.act_quant_fp8(x, pow2=pow2)
    wq, ws = R.quantised(x, pow2)
    assert torch.equal(s.cpu(), ws)
    same_codes(torch, q, wq)


@pytest.mark.parametrize("pow2", (False, True))
def test_act_quant_values(torch, pow2):
    """Zeros, tiny and huge blocks, ties, NaN and infinities; pitched and unaligned rows."""
    from ainfer_amd import moe
    x = torch.randn(12, 400, generator=gen(torch, 3), device="cuda")
    x[0] = 0
    x[1] *= 1e-44
    x[2] *= 1e-38
    x[3] *= 1e37
    x[4] = 3.4e38
    x[5] = torch.arange(400, device="cuda") / 16.0   # many ties
    x[6, 5] = float("nan")
    x[7, 130] = float("inf")
    x[8, 399] = -float("inf")
    x[9] = -0.0
    x[10, :128] = float("nan")
    x[11] = torch.exp2(torch.randint(-30, 30, (400,), device="cuda").float())
    for src in (x, x.to(torch.bfloat16)):
        wq, ws = R.quantised(src, pow2)
        for pad, off in ((0, 0), (7, 0), (9, 3)):
            buf = torch.zeros(12, 400 + pad + off, device="cuda", dtype=src.dtype)
            view = buf[:, off:off + 400]
            view.copy_(src)
            q = torch.full((12, 432), 7.0, device="cuda").to(R.E4M3)
            s = torch.empty(12, 4, device="cuda")
            moe.act_quant_fp8(view, q[:, :400], s, pow2=pow2)
            assert torch.equal(s.cpu(), ws)
            same_codes(torch, q[:, :400], wq)
            assert (q[:, 400:].float() == 7).all()


@pytest.mark.parametrize("pow2", (False, True))
def test_act_quant_next_to_ties(torch, pow2):
    """Values next to the borders between codes: a quotient that is off by one unit of the
    last place takes the other code."""
    from ainfer_amd import moe
    g = torch.Generator().manual_seed(11)
    n = 4000
    most = torch.exp2(torch.rand(n, generator=g) * 200 - 130) * (1 + torch.rand(n, generator=g))
    s = R.scale_of(most, pow2)
    codes = torch.arange(0x7F, dtype=torch.uint8).view(R.E4M3).double()  # 0 to 448
    border = (codes[:-1] + codes[1:]) / 2
    near = (border * s.double()[:, None]).float()                        # [n][126]
    sign = torch.where(torch.rand(n, 126, generator=g) < 0.5, -1.0, 1.0)
    up = torch.nextafter(near, torch.full_like(near, 3e38))
    down = torch.nextafter(near, torch.zeros_like(near))
    rows = torch.cat([torch.cat([most[:, None], t * sign, most[:, None]], 1) for t in (near, up, down)], 1)
    rows = rows.clamp(-most[:, None], most[:, None])
    wq, ws = R.quantised(rows, pow2)
    q, sq = moe.act_quant_fp8(rows.cuda(), pow2=pow2)
    assert torch.equal(sq.cpu(), ws)
    same_codes(torch, q, wq)


def test_act_quant_quotients_next_to_half_units(torch):
    """Small scales and quotients a few 2^-24ths of a unit from half a unit above a border
    between two codes: a quotient rounded the other way is the border itself and takes the
    even code.  v = (S h - j 2^-24) units for scales of S units, h the border plus half a unit
    of its last place, 2^24 h = A: S = j / A modulo 2^24."""
    from ainfer_amd import moe
    rows = []
    for power in (-103, -100, -99, -98, -97, -94, -91, -89):
        for num in (1, 3, 5, 7, 9, 11, 13, 15):                       # border num / 1024
            high = num.bit_length() - 1
            A = (num << 24 >> high) + 1
            for j in range(-200, 201):
                S = j * pow(A, -1, 1 << 24) % (1 << 24)
                if S < 1 << 23:
                    continue
                V = (S * A - j) >> 24
                s, v = (x * 2.0 ** (power - 23) for x in (S, V * 2.0 ** (high - 10)))
                most = torch.tensor(448 * s, dtype=torch.float32)
                if V < 1 << 24 and (most / 448).item() == s:
                    rows.append([most.item(), v, -v, 0.0] * 4)
    rows = torch.tensor(rows, dtype=torch.float64).float()
    assert len(rows) > 1000
    wq, ws = R.quantised(rows, False)
    q, sq = moe.act_quant_fp8(rows.cuda())
    assert torch.equal(sq.cpu(), ws)
    same_codes(torch, q, wq)


@pytest.mark.parametrize("pow2", (False, True))
@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("n,I", ((1, 16), (3, 144), (128, 512), (70, 1040), (1000, 128)))
def test_silu_mul_fp8(torch, n, I, dtype, pow2):
    from ainfer_amd import moe
    g = gen(torch, n + I)
    gu = (torch.randn(n, 2 * I + 3, generator=g, device="cuda") * 2).to(getattr(torch, dtype))
    gate, up = gu[:, :I], gu[:, I:2 * I]
    q, s = moe.silu_mul_fp8(gate, up, pow2=pow2)
    v = gate.double() * torch.sigmoid(gate.double()) * up.double()
    m = torch.nn.functional.pad(v, (0, -I % 128)).view(n, -1, 128).abs().amax(2) / R.TOP
    if pow2:
        assert (torch.frexp(s)[0] == 0.5).all()
        assert (s >= m * (1 - 2.0 ** -20)).all() and (s / 2 < m * (1 + 2.0 ** -20)).all()
    else:
        assert ((s - m).abs() <= 2.0 ** -20 * m).all()
    sw = R.wide(s.double(), 1, I)
    off = (q.double() * sw - v).abs()
    assert (off <= (2.0 ** -4 + 2.0 ** -20) * v.abs() + 2.0 ** -10 * sw * (1 + 2.0 ** -20)).all()


def test_silu_mul_fp8_of_far_gates(torch):
    """Gates whose exponential nears fp32's largest value or passes it: within 2^-119 of up
    beside the codes' rounding, and no infinities."""
    from ainfer_amd import moe
    n, I = 64, 256
    g = gen(torch, 3)
    gate = torch.linspace(-130, -70, n * I, device="cuda").view(n, I)
    for size in (1.0, 1e30, 1e-30):
        up = torch.randn(n, I, generator=g, device="cuda") * size
        q, s = moe.silu_mul_fp8(gate, up)
        v = gate.double() * torch.sigmoid(gate.double()) * up.double()
        sw = R.wide(s.double(), 1, I)
        off = (q.double() * sw - v).abs()
        bound = (2.0 ** -4 + 2.0 ** -20) * v.abs() + 2.0 ** -10 * sw * (1 + 2.0 ** -20)
        assert s.isfinite().all() and (off <= bound + 2.0 ** -119 * up.double().abs()).all()
    far = torch.tensor([-3e38, -1e4, -200.5, 3e38, 1e4, 0.0, -0.0, float("inf")] * 16, device="cuda")
    q, s = moe.silu_mul_fp8(far[None], torch.full_like(far, 0.5)[None])
    assert s.isinf().all()  # the infinite gate's
    q, s = moe.silu_mul_fp8(far[None, :112].where(far[:112].isfinite(), torch.zeros(())), torch.ones(
        1, 112, device="cuda"))
    assert s.isfinite().all() and (q.float() * s[0, 0] <= 3.1e38).all() and q.float().max() == 448


def test_live_rows(torch):
    """Rows behind the count, and columns behind the row, are left as they are."""
    from ainfer_amd import moe
    x = torch.randn(20, 272, generator=gen(torch, 8), device="cuda")
    for live in (-3, 0, 1, 13, 20, 25):
        count = torch.tensor([9, 9, live], dtype=torch.int32, device="cuda")
        keep = max(0, min(live, 20))
        for call in (lambda q, s: moe.act_quant_fp8(x, q, s, live=count),
                     lambda q, s: moe.silu_mul_fp8(x, x, q, s, live=count)):
            q = torch.full((20, 272), 2.0, device="cuda").to(R.E4M3)
            s = torch.full((20, 3), -5.0, device="cuda")
            call(q, s)
            assert (q[keep:].float() == 2).all() and (s[keep:] == -5).all()
            assert (s[:keep] > 0).all()
        d = [torch.full((20, 272), 3.0, device="cuda") for _ in range(2)]
        moe.silu_mul_backward(x, x, x, *d, live=count)
        for t in d:
            assert (t[keep:] == 3).all() and not (t[:keep] == 3).any()


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("E,M,K", ((1, 1, 16), (1, 128, 128), (2, 130, 144), (3, 300, 400), (2, 64, 2048)))
def test_weight_quant(torch, E, M, K, dtype):
    from ainfer_amd import moe
    for pow2 in (False, True):
        w = torch.randn(E, M, K, generator=gen(torch, M + K), device="cuda").to(getattr(torch, dtype))
        w[0, 0, 0] = 0
        q, scales = moe.weight_quant_fp8(w, pow2=pow2)
        b = torch.nn.functional.pad(w.float().cpu(), (0, -K % 128, 0, -M % 128))
        b = b.view(E, R.groups(M), 128, R.groups(K), 128)
        s = R.scale_of(b.abs().amax((2, 4)), pow2)
        assert torch.equal(scales.cpu(), s)
        want = (b / s[:, :, None, :, None]).reshape(E, R.groups(M) * 128, -1)[:, :M, :K]
        same_codes(torch, q, want.to(R.E4M3))


@pytest.mark.parametrize("E,M,K", ((1, 1, 16), (2, 64, 128), (3, 130, 144), (1, 65, 272), (2, 304, 400)))
def test_pack(torch, E, M, K):
    """Tiles of 64 x 128: tile i's row r is row 32 (i / 2) + 8 (r / 4) + 4 (i % 2) + r % 4, two
    halves of 64 columns, 16 of each quarter to lane 16 quarter + r; zeros behind the matrix."""
    from ainfer_amd import _lib as L
    from ainfer_amd import moe
    w = torch.randint(0, 256, (E, M, K), device="cuda", dtype=torch.uint8)
    mb, G = -(-M // 64), R.groups(K)
    full = torch.zeros(E, mb * 64, G * 128, dtype=torch.uint8, device="cuda")
    full[:, :M, :K] = w
    # [e][mb][i / 2][r / 4][i % 2][r % 4][g][half][quarter][16]
    #   -> [e][mb][g][i][half][quarter][r][16]
    want = full.view(E, mb, 2, 4, 2, 4, G, 2, 4, 16).permute(0, 1, 6, 2, 4, 7, 8, 3, 5, 9).reshape(-1)
    f = moe.Fp8Weights(w, torch.ones(E, R.groups(M), G, device="cuda"))
    assert f.packed.numel() == want.numel() == L.lib().ainfer_moe_fp8_packed_bytes(E, M, K)
    assert torch.equal(f.packed, want)
    t = w.transpose(1, 2).contiguous()
    s = torch.rand(E, G, R.groups(M), device="cuda")
    b = moe.Fp8Weights(t, s, transpose=True)
    assert torch.equal(b.packed, want) and torch.equal(b.scales, s.transpose(1, 2))
    assert b.shape == (E, M, K)


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("n,I,pad", ((1, 1, 0), (3, 7, 0), (5, 64, 3), (100, 333, 1), (1000, 512, 0)))
def test_silu_backward(torch, n, I, pad, dtype):
    """Against the formula in 64 bits: sig to 2^-21, 1 - sig to 2^-21 absolutely, so the
    bracket is off by (1 + |g|) 2^-20 at most; and against differences."""
    from ainfer_amd import moe
    dt = getattr(torch, dtype)
    g = gen(torch, n + I)
    gu = (torch.randn(n, 2 * I + pad, generator=g, device="cuda") * 3).to(dt)
    gate, up = gu[:, :I], gu[:, I:2 * I]
    d = torch.randn(n, I, generator=g, device="cuda").to(dt)
    out = torch.full((n, 2 * I + pad), 9.0, device="cuda", dtype=dt)
    moe.silu_mul_backward(d, gate, up, out[:, :I], out[:, I:2 * I])
    assert (out[:, 2 * I:] == 9).all()
    dd, gg, uu = d.double(), gate.double(), up.double()
    sig = torch.sigmoid(gg)
    half = 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -24
    want = dd * uu * sig * (1 + gg * (1 - sig))
    off = (out[:, :I].double() - want).abs()
    assert (off <= (dd * uu).abs() * sig * (1 + gg.abs()) * 2.0 ** -20 + half * want.abs()
            * (1 + 2.0 ** -8) + 1e-37).all()
    want = dd * gg * sig
    off = (out[:, I:2 * I].double() - want).abs()
    assert (off <= (2.0 ** -20 + half) * want.abs() + 1e-37).all()
    h = 1e-5
    f = lambda a: a * torch.sigmoid(a) * uu * dd  # noqa: E731
    slope = (f(gg + h) - f(gg - h)) / (2 * h)
    assert (out[:, :I].double() - slope).abs().max() <= (half + 1e-4) * slope.abs().max() + 1e-6


def test_silu_backward_in_place_and_extremes(torch):
    from ainfer_amd import moe
    x = [torch.randn(9, 40, generator=gen(torch, 5), device="cuda") for _ in range(3)]
    want = [torch.empty_like(x[0]) for _ in range(2)]
    moe.silu_mul_backward(*x, *want)
    for a, b in ((0, 1), (1, 2), (2, 0), (1, 0)):
        y = [t.clone() for t in x]
        moe.silu_mul_backward(*y, y[a], y[b])
        assert torch.equal(y[a], want[0]) and torch.equal(y[b], want[1])
    g = torch.tensor([[100.0, -100.0, 3e38, -3e38, 0.0]], device="cuda")
    one = torch.ones_like(g)
    moe.silu_mul_backward(one, g, one, a := torch.empty_like(g), b := torch.empty_like(g))
    assert a[0].tolist()[:1] == [1.0] and abs(a[0, 1]) < 1e-37 and a[0, 2] == 1 and a[0, 3] == 0
    assert a[0, 4] == 0.5 and b[0].tolist()[::2] == [100.0, g[0, 2].item(), 0.0]


# ---- products -------------------------------------------------------------------

def state(torch, counts, M, K, seed, pad=(0, 0), extra=0):
    """Rows of each expert, `extra` rows behind the last one's."""
    g = gen(torch, seed)
    E, n = len(counts), sum(counts) + extra
    q = R.codes(g, n, K + pad[0])[:, :K]
    sq = torch.rand(n, R.groups(K), generator=g, device="cuda") / 100 + 1e-3
    w = R.codes(g, E, M, K)
    scales = torch.rand(E, R.groups(M), R.groups(K), generator=g, device="cuda") / 100 + 1e-3
    offsets = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32,
                           device="cuda")
    return q, sq, w, scales, offsets


def check(torch, q, sq, w, scales, offsets, dtype, y=None, seed=1):
    from ainfer_amd import moe
    n, M, K = q.shape[0], w.shape[1], q.shape[1]
    print(f"[case] product {n} x {K} -> {M}, {w.shape[0]} experts, {dtype}", flush=True)
    if y is None:
        y = torch.randn(n, M, generator=gen(torch, seed), device="cuda").to(dtype)
    before = y.clone()
    want, size = R.product(q, sq, w, scales, offsets, before)
    moe.Fp8Weights(w, scales).product(q, sq, y, offsets)
    torch.cuda.synchronize()
    bound = (128 + R.groups(K) + 4) * 2.0 ** -24 * size
    if dtype == torch.bfloat16:
        bound = (bound + 7 * 2.0 ** -13 * size) * 1.01 + 2.0 ** -8 * want.abs() * (size > 0)
    else:
        bound = bound + 2.0 ** -24 * want.abs() * (size > 0)
    off = (y.double() - want).abs()
    if dtype == torch.bfloat16 and n * M > 1000:
        assert off.norm() <= (2.0 ** -8 + 2.0 ** -11) * want.norm()
    assert (off <= bound).all(), (off - bound).max().item()
    return y


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("n,M,K", ((1, 1, 16), (1, 16, 128), (1, 130, 144), (2, 333, 2048),
                                   (16, 256, 512), (17, 300, 400), (63, 128, 1040), (64, 1000, 256),
                                   (128, 256, 384), (129, 257, 272), (300, 513, 640),
                                   (1000, 640, 2048), (5, 17408, 256), (3, 64, 65536)))
def test_product_dense(torch, n, M, K, dtype):
    q, sq, w, scales, offsets = state(torch, [n], M, K, n + M + K)
    dt = getattr(torch, dtype)
    a = check(torch, q, sq, w, scales, offsets, dt)
    b = check(torch, q, sq, w, scales, None, dt)
    assert torch.equal(a, b)


COUNTS = ([1, 0, 3], [0, 0, 0, 1], [5, 17, 0, 16, 1], [128, 129, 127], [1] * 40, [0, 300, 0, 2],
          [64] * 9, [31, 33, 65, 257, 0, 1], [2] * 300)


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("M,K", ((130, 272), (256, 512), (515, 1040)))
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}e{sum(c)}")
def test_product_grouped(torch, counts, M, K, dtype):
    q, sq, w, scales, offsets = state(torch, counts, M, K, sum(counts) + M, extra=7)
    check(torch, q, sq, w, scales, offsets, getattr(torch, dtype))


def spread(seed, E, most):
    """Rows of E experts: none for some, 1, 15, 16, 17 and every other number up to most."""
    import random
    r = random.Random(seed)
    some = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, most]
    return [r.choice(some) if r.random() < 0.3 else r.randint(0, most) for _ in range(E)]


# (rows of each expert, M, K): large enough for the tiled forms.  128 rows a tile and one group
# of weights ahead from 200 tiles on, else 96 and two (bf16); 96 rows and one from 600 tiles on,
# else 64 and two (fp32); K of one to six groups, whole and not
TILED = tuple((spread(K, 64, 300), M, K) for M in (1030, 2100)
              for K in (16, 128, 144, 256, 400, 512, 640, 752)) + (
    ([5000], 7000, 272), ([5000], 7001, 128), ([1, 4000, 0, 1000], 7000, 400),
    ([64] * 40 + [0] * 30 + [200] * 30, 1030, 384), ([2000, 3], 4100, 2048), ([7] * 300, 1500, 272),
    ([0] * 500 + [3000] + [0] * 523, 2049, 272), ([40] * 1024, 300, 144)) + tuple(
    (spread(K + 1, E, total), M, K) for E, total, M in ((64, 3000, 1030), (20, 200, 700))
    for K in (16, 128, 144, 256, 400, 512, 640, 752))


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("case", range(len(TILED)))
def test_product_tiled(torch, case, dtype):
    counts, M, K = TILED[case]
    q, sq, w, scales, offsets = state(torch, counts, M, K, case, pad=(16, 0), extra=5)
    # NaN codes between pitched rows, behind the last row and in what no expert holds
    base = q.as_strided((q.shape[0], K + 16), (K + 16, 1)).view(torch.uint8)
    base[:, K:] = 0x7F
    base[-5:] = 0x7F
    sq[-5:] = float("nan")
    y = check(torch, q, sq, w, scales, offsets, getattr(torch, dtype))
    again = y.clone().fill_(3)
    from ainfer_amd import moe
    moe.Fp8Weights(w, scales).product(q, sq, again, offsets)
    n = int(offsets[-1])
    assert torch.equal(again[:n], y[:n]) and (again[n:] == 3).all()


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
def test_product_pitches(torch, dtype):
    """Pitched codes and outputs, outputs that start at odd elements; other columns stay."""
    dt = getattr(torch, dtype)
    for counts in ([3, 0, 2], [40, 90, 200]):
        for M, off in ((130, 0), (131, 1), (256, 3)):
            q, sq, w, scales, offsets = state(torch, counts, M, 400, 77, pad=(48, 0), extra=5)
            buf = torch.full((q.shape[0], M + 6), 3.0, device="cuda", dtype=dt)
            check(torch, q, sq, w, scales, offsets, dt, y=buf[:, off:off + M])
            assert (buf[:, :off] == 3).all() and (buf[:, off + M:] == 3).all()


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
def test_product_largest_pitch(torch, dtype):
    """Rows of codes 2^24 bytes apart: a tile's last one is 2^31 - 2^24 behind its first."""
    for M in (200, 30000):
        q, sq, w, scales, offsets = state(torch, [130], M, 272, M)
        far = torch.empty((129 << 24) + 272, dtype=torch.uint8, device="cuda").view(R.E4M3)
        far = far.as_strided((130, 272), (1 << 24, 1))
        far.copy_(q)
        check(torch, far, sq, w, scales, offsets, getattr(torch, dtype))


def test_product_garbage_behind_the_row(torch):
    """NaN codes in the padding of pitched rows and in the next row's weights change nothing."""
    for counts in ([2, 1], [70, 60]):
        q, sq, w, scales, offsets = state(torch, counts, 100, 144, 5, pad=(16, 0))
        base = q.as_strided((q.shape[0], 160), (160, 1))
        base[:, 144:].view(torch.uint8).fill_(0x7F)
        y = check(torch, q, sq, w, scales, offsets, torch.float32)
        assert y.isfinite().all()


def test_product_nan_stays_in_its_row(torch):
    for counts in ([2, 1], [70, 60], [400, 300]):
        q, sq, w, scales, offsets = state(torch, counts, 300, 272, 6)
        q = q.contiguous()
        from ainfer_amd import moe
        y = moe.Fp8Weights(w, scales).product(q, sq, offsets=offsets, y=torch.empty(len(q), 300, device="cuda"))
        bad = q.clone()
        bad.view(torch.uint8)[1, 200] = 0xFF
        z = moe.Fp8Weights(w, scales).product(bad, sq, offsets=offsets, y=torch.empty(len(q), 300, device="cuda"))
        assert z[1].isnan().all()
        keep = torch.arange(len(q), device="cuda") != 1
        assert torch.equal(z[keep], y[keep])


def test_product_offsets_out_of_range(torch):
    """Offsets outside [0, N] are its ends: no row outside is touched."""
    from ainfer_amd import moe
    q, sq, w, scales, _ = state(torch, [20, 20], 130, 256, 9)
    buf = torch.full((60, 130), 4.0, device="cuda")
    offsets = torch.tensor([-5, 1000, 1 << 30], dtype=torch.int32, device="cuda")
    moe.Fp8Weights(w, scales).product(q, sq, buf[10:50], offsets)
    assert (buf[:10] == 4).all() and (buf[50:] == 4).all() and not (buf[10:50] == 4).all(1).any()


def test_product_streams_and_graph(torch):
    """On another stream, and captured: replays equal eager calls on the inputs of then."""
    from ainfer_amd import moe
    for counts in ([3, 0, 2], [200, 300]):
        q, sq, w, scales, offsets = state(torch, counts, 256, 512, 21)
        f = moe.Fp8Weights(w, scales)
        want = f.product(q, sq, offsets=offsets)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = f.product(q, sq, offsets=offsets, stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        y = torch.zeros_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f.product(q, sq, y, offsets)
        for i in range(4):
            q.copy_(R.codes(gen(torch, 100 + i), *q.shape))
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, f.product(q, sq, offsets=offsets))


def test_product_large_addresses(torch):
    """Weights of more than 2^32 bytes, codes and outputs of more than 2^31 elements."""
    from ainfer_amd import moe
    E, M, K = 300, 3968, 4096
    w = torch.randint(0, 120, (E, M, K), device="cuda", dtype=torch.uint8).view(R.E4M3)
    scales = torch.rand(E, 31, 32, device="cuda") + 0.5
    counts = [0] * E
    counts[0], counts[E - 1], counts[E - 2] = 3, 5, 200
    q, sq, _, _, offsets = state(torch, counts, 16, K, 3)
    y = moe.Fp8Weights(w, scales).product(q, sq, offsets=offsets)
    for e in (0, E - 2, E - 1):
        a, b = int(offsets[e]), int(offsets[e + 1])
        want, size = R.product(q[a:b], sq[a:b], w[e:e + 1], scales[e:e + 1], None,
                               torch.zeros(b - a, M, device="cuda"))
        assert ((y[a:b].double() - want).abs() <= 7.1 * 2.0 ** -13 * size + 2.0 ** -7.9 * want.abs()).all()
    del w, y
    N, K, M = 300000, 7552, 7424
    q = torch.randint(0, 120, (N, K), device="cuda", dtype=torch.uint8).view(R.E4M3)
    sq = torch.rand(N, 59, device="cuda") + 0.5
    w, scales = R.codes(gen(torch, 1), 1, M, K), torch.rand(1, 58, 59, device="cuda") + 0.5
    y = moe.Fp8Weights(w, scales).product(q, sq)
    for r in (0, 150000, N - 1):
        want, size = R.product(q[r:r + 1], sq[r:r + 1], w, scales, None, torch.zeros(1, M, device="cuda"))
        assert ((y[r:r + 1].double() - want).abs() <= 7.1 * 2.0 ** -13 * size + 2.0 ** -7.9 * want.abs()).all()
