"""Plain 64-bit forms of the 8-bit floating point operators, for their tests."""
import torch

TOP = 448.0
E4M3 = torch.float8_e4m3fn


def groups(n):
    return -(-n // 128)


def wide(scales, dim, n):
    """Each block's scale at the values that it stands for."""
    return scales.repeat_interleave(128, dim).narrow(dim, 0, n)


def scale_of(m, pow2):
    """The scale of blocks of largest magnitude m (fp32, IEEE operations)."""
    s = (m / TOP).clamp_min(2.0 ** -126)
    if pow2:
        f, e = torch.frexp(s)
        s = torch.where(s.isinf(), s, torch.ldexp(torch.ones_like(s), e - (f == 0.5).to(torch.int32)))
    return torch.where(m == 0, torch.ones_like(s), s)


def quantised(x, pow2):
    """(codes, scales) of the rows of x by the definition, bit for bit (on the CPU)."""
    x = x.float().cpu()
    n, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % 128)).view(n, -1, 128)
    m = torch.where(b.isnan(), torch.zeros_like(b), b.abs()).amax(2)
    s = scale_of(m, pow2)
    return (b / s[:, :, None]).reshape(n, -1)[:, :K].to(E4M3), s


def codes(g, *shape, std=100.0):
    """Random codes, some of them the largest and the smallest values."""
    x = torch.randn(*shape, generator=g, device="cuda").mul_(std).clamp_(-TOP, TOP)
    return x.to(E4M3)


def product(q, sq, w, scales, offsets, y):
    """(values, sums of magnitudes) of ainfer_moe_fp8_product's rows, in 64 bits; y's own
    rows outside the offsets."""
    K, M = q.shape[1], w.shape[1]
    out = y.double().clone()
    size = torch.zeros_like(out)
    x = q.double() * wide(sq.double(), 1, K)
    bounds = [0, q.shape[0]] if offsets is None else offsets.tolist()
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if b > a:
            we = w[e].double() * wide(wide(scales[e].double(), 1, K), 0, M)
            out[a:b] = x[a:b] @ we.t().contiguous()
            size[a:b] = x[a:b].abs() @ we.abs().t().contiguous()
    return out, size


def sort(idx, E):
    """(offsets, pos, pair of each kept row) on the CPU."""
    ids = idx.cpu().reshape(-1).tolist()
    by = [[] for _ in range(E)]
    for i, e in enumerate(ids):
        if 0 <= e < E:
            by[e].append(i)
    offsets = [0]
    for b in by:
        offsets.append(offsets[-1] + len(b))
    order = [i for b in by for i in b]
    pos = torch.full((len(ids),), -1, dtype=torch.int32)
    if order:
        pos[torch.tensor(order)] = torch.arange(len(order), dtype=torch.int32)
    return torch.tensor(offsets, dtype=torch.int32), pos.view(idx.shape), order
