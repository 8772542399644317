"""Adapters of many requests (ainfer_moe_lora_apply) against the formula in 64 bits.

Bound per element, from the arithmetic: x and A enter exactly and v is a sum of K
products in fp32, so |v - v64| <= (K + 32) 2^-23 sum|x||A| (2^-23: the matrix
instructions may round either way); v * scale rounds once; as two bf16 parts (y in
bf16) it is off by 2^-16, as three not at all; the second sum has at most 3 R terms;
y rounds once (2^-24, or 2^-8 in bf16)."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


class Case:
    def __init__(self, torch, T, N, R, K, Ms, x="bf16", y="fp32", ids=None, ranks=None,
                 scales=True, seed=0, x_pad=0, y_pad=0):
        dt = {"bf16": torch.bfloat16, "fp32": torch.float32}
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + T * 31 + K)

        def normal(*s, std=1.0, dtype=torch.float32):
            return (torch.randn(*s, generator=g, device="cuda") * std).to(dtype)

        self.torch, self.T, self.N, self.R, self.K, self.Ms = torch, T, N, R, K, Ms
        self.a = [normal(N, R, K, std=K ** -0.5, dtype=torch.bfloat16) for _ in Ms]
        self.b = [normal(N, M, R, std=0.2, dtype=torch.bfloat16) for M in Ms]
        self.x = normal(T, K + x_pad, dtype=dt[x])[:, :K]
        self.y = [normal(T, M + y_pad, dtype=dt[y])[:, :M] for M in Ms]
        self.scales = torch.rand(N, generator=g, device="cuda") + 0.5 if scales else None
        if ranks is None:
            self.ranks = None
        else:
            self.ranks = torch.tensor(ranks, dtype=torch.int32, device="cuda")
        if ids is None:
            ids = torch.randint(-1, N, (T,), generator=g, device="cuda").tolist()
        self.ids = torch.tensor(ids, dtype=torch.int32, device="cuda")
        from ainfer_amd.moe import LoraAdapters
        self.lora = LoraAdapters(self.a, self.b, ranks=self.ranks, scales=self.scales,
                                 x_dtype=dt[x], y_dtype=dt[y])
        print(f"[case] T={T} N={N} R={R} K={K} M={Ms} x={x} y={y}", flush=True)

    def apply(self, ys, ws=None, stream=None):
        ws = self.lora.workspace(self.T) if ws is None else ws
        self.lora.apply(self.x, self.ids, ys, ws, stream=stream)

    def check(self):
        torch = self.torch
        ys = [y.clone() if y.is_contiguous() else y for y in self.y]
        before = [y.clone() for y in ys]
        self.apply(ys)
        torch.cuda.synchronize()
        self.compare(before, ys)

    def compare(self, before, after):
        torch = self.torch
        step = 2.0 ** -24 if before[0].dtype == torch.float32 else 2.0 ** -8
        split = 0.0 if before[0].dtype == torch.float32 else 2.0 ** -16
        ids = self.ids.cpu()
        for p in range(len(self.Ms)):
            y0, y1 = before[p].double().cpu(), after[p].double().cpu()
            want, bound = y0.clone(), torch.zeros_like(y0)
            same = torch.ones(self.T, dtype=torch.bool)
            x = self.x.double().cpu()
            for n in sorted(set(ids.tolist())):
                if not 0 <= n < self.N:
                    continue
                r = self.R
                if self.ranks is not None:
                    r = min(max(int(self.ranks[n]), 0), self.R)
                rows = (ids == n).nonzero()[:, 0]
                if r == 0:
                    continue
                same[rows] = False
                s = 1.0 if self.scales is None else float(self.scales[n])
                A = self.a[p][n, :r].double().cpu()
                B = self.b[p][n, :, :r].double().cpu()
                v = x[rows] @ A.t()
                mag = x[rows].abs() @ A.abs().t()
                want[rows] += s * (v @ B.t())
                bound[rows] = s * (((self.K + 3 * self.R + 40) * 2.0 ** -23 * mag
                                    + split * v.abs()) @ B.abs().t())
            assert torch.equal(y1[same], y0[same])       # rows without an adapter: untouched
            assert torch.isfinite(y1).all()
            assert ((y1 - want).abs() <= bound * (1 + step) + step * want.abs()).all(), (
                p, float(((y1 - want).abs() - bound - step * want.abs()).max()))


# T, N, R, K, Ms: one token, odd token counts around the tile sizes, ranks of every
# block count, K of one chunk to many with tails, M of one to many with tails
SHAPES = [(1, 1, 8, 8, [1]), (1, 4, 16, 4096, [4096]), (2, 3, 8, 72, [33, 7]),
          (5, 2, 24, 520, [100]), (16, 16, 64, 1024, [257]), (17, 5, 32, 200, [64, 64, 31]),
          (63, 40, 16, 640, [96]), (64, 64, 128, 264, [40]), (65, 3, 40, 136, [129]),
          (255, 9, 16, 264, [48, 80]), (257, 7, 8, 128, [65]), (300, 2, 104, 328, [72]),
          (1003, 12, 8, 1024, [136, 1, 2, 3]), (40, 2, 96, 2056, [33]),
          (129, 3, 32, 2184, [1100, 260]), (700, 5, 64, 1096, [64]), (150, 20, 40, 72, [131]),
          (1030, 2, 128, 520, [516]), (513, 1, 24, 8, [4])]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("x,y", (("bf16", "fp32"), ("fp32", "bf16"), ("fp32", "fp32"),
                                 ("bf16", "bf16")))
def test_matches_formula(torch, shape, x, y):
    Case(torch, *shape, x=x, y=y).check()


@pytest.mark.parametrize("R", (8, 16, 24, 32, 64, 72, 128))
@pytest.mark.parametrize("T", (50, 200))
def test_ragged_ranks_and_garbage_beyond_them(torch, R, T):
    """Ranks 0, 1, odd ones, R, and values outside 0..R; NaN and inf in the rows
    of A and columns of B beyond them."""
    ranks = [0, 1, 3, R - 1, R, -4, R + 9, R // 2]
    c = Case(torch, T, 8, R, 136, [72, 9], ranks=ranks)
    for n, r in enumerate(ranks):
        r = min(max(r, 0), R)
        for a, b in zip(c.a, c.b):
            a[n, r:] = math.nan
            b[n, :, r:] = math.inf
    c.check()


@pytest.mark.parametrize("T", (1, 20, 100, 700))
def test_prompts_and_tokens_without_adapter(torch, T):
    """Requests one after the other, ids outside the adapters, all without one."""
    ids = [(t * 5 // T) - 1 for t in range(T)]
    Case(torch, T, 4, 16, 264, [100], ids=ids).check()
    Case(torch, T, 4, 16, 264, [100], ids=[4] * T, y="bf16").check()
    Case(torch, T, 4, 16, 264, [100], ids=[(-7, 4, 1 << 30)[t % 3] for t in range(T)]).check()
    Case(torch, T, 4, 16, 264, [100], ids=[t % 4 for t in range(T)], scales=False).check()


def test_pitches_and_alignment(torch):
    """Rows of x and y inside wider ones: 16-byte pieces of y, and not."""
    for y in ("fp32", "bf16"):
        for pad in (8, 3, 1):
            for T, R in ((33, 16), (150, 8), (150, 32), (140, 128)):
                Case(torch, T, 5, R, 200, [64, 50], x_pad=8, y_pad=pad, y=y).check()
                Case(torch, T, 5, R, 200, [68], x_pad=8, y_pad=pad, y=y, x="fp32").check()


@pytest.mark.parametrize("T", (32, 160))
def test_other_tokens_do_not_leak(torch, T):
    """A token's NaN and an adapter's inf stay in that token's rows and that
    adapter's tokens."""
    c = Case(torch, T, 4, 16, 264, [80], ids=[t % 4 for t in range(T)])
    c.x[5] = math.nan
    c.b[0][3] = math.inf
    ys = [y.clone() for y in c.y]
    c.apply(ys)
    torch.cuda.synchronize()
    bad = torch.tensor([t == 5 or t % 4 == 3 for t in range(T)], device="cuda")
    assert not torch.isfinite(ys[0][bad]).any()
    assert torch.isfinite(ys[0][~bad]).all()
    d = Case(torch, T, 4, 16, 264, [80], ids=[t % 4 for t in range(T)])
    clean = [y.clone() for y in d.y]
    d.apply(clean)
    assert torch.equal(clean[0][~bad], ys[0][~bad])


@pytest.mark.parametrize("T", (4, 140))
def test_infinite_and_large_fp32_inputs(torch, T):
    """fp32 x of inf gives inf, the largest finite x what the formula gives."""
    c = Case(torch, T, 1, 8, 64, [16], x="fp32", ids=[0] * T, ranks=[1], scales=False)
    c.a[0].zero_()
    c.a[0][:, 0, 0] = 1.0
    c.b[0].zero_()
    c.b[0][:, :, 0] = 2.0 ** -10
    c.x.zero_()
    c.x[0, 0] = math.inf
    c.x[1, 0] = torch.finfo(torch.float32).max
    c.x[2, 0] = 1 + 2.0 ** -23
    ys = [torch.zeros_like(c.y[0])]
    c.apply(ys)
    torch.cuda.synchronize()
    assert (ys[0][0] == math.inf).all()
    assert (ys[0][1] == torch.finfo(torch.float32).max * 2.0 ** -10).all()
    assert (ys[0][2] == (1 + 2.0 ** -23) * 2.0 ** -10).all()
    assert (ys[0][3] == 0).all()


def test_shared_workspace_streams_and_graph(torch):
    """One workspace for calls of several sizes in turn; another stream; a captured
    call replayed between eager ones."""
    big = Case(torch, 300, 6, 16, 520, [200])
    ws = big.lora.workspace(300)
    for T in (300, 1, 17, 300):
        c = Case(torch, T, 6, 16, 520, [200], seed=T)
        ys = [y.clone() for y in c.y]
        c.apply(ys, ws)
        torch.cuda.synchronize()
        c.compare(c.y, ys)
    side = torch.cuda.Stream()
    ys = [y.clone() for y in big.y]
    side.wait_stream(torch.cuda.current_stream())
    big.apply(ys, ws, stream=side)
    side.synchronize()
    big.compare(big.y, ys)
    ref = [y.clone() for y in ys]
    buf = [y.clone() for y in big.y]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        big.apply(buf, ws)
    for _ in range(3):
        for b, y in zip(buf, big.y):
            b.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(b, r) for b, r in zip(buf, ref))
        Case(torch, 17, 6, 16, 520, [200]).check()


@pytest.mark.parametrize("T,pitch", ((33, (1 << 27) + 8), (130, (1 << 26) + (1 << 23)),
                                     (200, (1 << 24) + 8)))
def test_offsets_past_32_bits(torch, T, pitch):
    """x and y pitches whose products with the token pass 2^31 elements, or
    2^31 bytes within 16 tokens."""
    K, M = 64, 48
    c = Case(torch, T, 3, 8, K, [M])
    xs = torch.empty((T - 1) * pitch + K, dtype=torch.bfloat16, device="cuda")
    ys = torch.empty((T - 1) * pitch + M, dtype=torch.float32, device="cuda")
    x = xs.as_strided((T, K), (pitch, 1))
    y = ys.as_strided((T, M), (pitch, 1))
    x.copy_(c.x)
    y.copy_(c.y[0])
    c.lora.apply(x, c.ids, [y], c.lora.workspace(T))
    torch.cuda.synchronize()
    c.compare(c.y, [y.contiguous()])


# prompts whose A is read once, in a launch of its own: long K, ranks above 32
TWO_LAUNCHES = [(300, 7, 64, 4096, [1027]), (300, 3, 40, 4104, [1100, 1030]),
                (513, 2, 72, 2056, [1500]), (600, 4, 128, 1032, [2100]),
                (401, 5, 96, 4096, [640, 1300])]


@pytest.mark.parametrize("shape", TWO_LAUNCHES)
@pytest.mark.parametrize("x,y", (("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "bf16")))
def test_long_prompts_of_large_ranks(torch, shape, x, y):
    T, N, R = shape[:3]
    ids = [(t // 37) % (N + 1) - 1 if t < 200 else (t // 5) % N for t in range(T)]
    Case(torch, *shape, x=x, y=y, ids=ids).check()
    c = Case(torch, *shape, x=x, y=y, ids=ids, ranks=[(R - 9 * n) if n < 4 else 0 for n in range(N)])
    for n in range(N):                              # beyond a rank anything may stand
        r = max(int(c.ranks[n]), 0)
        for a, b in zip(c.a, c.b):
            a[n, r:] = float("nan")
            b[n, :, r:] = float("inf")
    c.check()


def test_workspace_of_pitched_prompts(torch):
    """More than 256 tokens at a pitch that the tiles' 32-bit offsets cannot
    reach, ranks that are not worth reading in every workgroup: one row of
    scratch per token.  Nothing past the workspace is written."""
    T, R, K, pitch = 300, 128, 1040, (1 << 26) + (1 << 23)
    c = Case(torch, T, 3, R, K, [48])
    xs = torch.empty((T - 1) * pitch + K, dtype=torch.bfloat16, device="cuda")
    c.x = xs.as_strided((T, K), (pitch, 1)).copy_(c.x)
    n = c.lora.workspace(T).numel()
    assert n >= T * R * 4
    buf = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    off = -buf.data_ptr() % 256
    ys = [y.clone() for y in c.y]
    c.apply(ys, buf[off:off + n])
    torch.cuda.synchronize()
    c.compare(c.y, ys)
    assert (buf[:off] == 0xA5).all() and (buf[off + n:] == 0xA5).all()


def test_two_launches_on_two_streams_and_in_a_graph(torch):
    """Calls at once on two streams, each with its own scratch; replays of a
    captured call with eager calls between them."""
    a = Case(torch, 300, 7, 64, 4096, [1027], seed=1)
    b = Case(torch, 411, 4, 96, 2048, [1500], x="fp32", seed=2)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    ys = [[y.clone() for y in c.y] for c in (a, b)]
    ws = [c.lora.workspace(c.T) for c in (a, b)]
    torch.cuda.synchronize()
    for c, y, w, s in zip((a, b), ys, ws, side):
        c.apply(y, w, stream=s)
    torch.cuda.synchronize()
    for c, y in zip((a, b), ys):
        c.compare(c.y, y)
    work = [y.clone() for y in a.y]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.apply(work, ws[0])
    for rep in range(3):
        for y, y0 in zip(work, a.y):
            y.copy_(y0)
        graph.replay()
        torch.cuda.synchronize()
        for y, want in zip(work, ys[0]):
            assert torch.equal(y, want), rep
        b.apply([y.clone() for y in b.y], ws[1])
        ws[0].fill_(rep)
        torch.cuda.synchronize()


@pytest.mark.parametrize("R", (8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128))
@pytest.mark.parametrize("x,y", (("bf16", "fp32"), ("bf16", "bf16"), ("fp32", "fp32"),
                                 ("fp32", "bf16")))
def test_prompts_of_every_rank(torch, R, x, y):
    """One launch and two, several chunks of K a wave, with and without the other."""
    Case(torch, 700, 3, R, 2312, [100], x=x, y=y).check()
    Case(torch, 290, 3, R, 4104, [70, 516], x=x, y=y, ids=[t // 60 % 4 - 1 for t in range(290)]).check()
    Case(torch, 1500, 3, R, 1160, [136], x=x, y=y).check()
    Case(torch, 330, 3, R, 1160, [2100], x=x, y=y).check()


@pytest.mark.parametrize("R", (8, 16, 24, 32, 40, 64, 72, 96, 120, 128))
@pytest.mark.parametrize("x,y", (("bf16", "fp32"), ("bf16", "bf16"), ("fp32", "fp32"),
                                 ("fp32", "bf16")))
def test_batches_of_every_rank(torch, R, x, y):
    Case(torch, 3, 2, R, 20488, [130], x=x, y=y, ids=[1, 0, 1]).check()
    Case(torch, 1, 2, R, 16384, [64, 1], x=x, y=y, ids=[1]).check()
    Case(torch, 41, 5, R, 2312, [70, 516], x=x, y=y).check()
    Case(torch, 200, 9, R, 1160, [100], x=x, y=y).check()
