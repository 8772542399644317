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
