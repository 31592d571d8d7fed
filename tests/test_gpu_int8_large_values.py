"""Rows of values near the largest of their type (masks of the lowest value among them): where a channel's scale makes the result finite, it is."""

import pytest
import torch

from oracle import int8 as oi

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _operands(m, k, n, dtype, groups=None):
    torch.manual_seed(m + n)
    x = torch.randn(m, k)
    most = 3e38 if dtype is not F16 else 65504.0
    x[::3] *= most / 8                                                       # no value of these rows is infinite: |x| < 6.5
    x[1::3, ::7] = -most
    x[2::6] = 0.0
    w = torch.randint(-127, 128, (*((groups,) if groups else ()), n, k), dtype=torch.int8, device="cuda")
    return x.clamp(-most, most).to(dtype).cuda(), w, torch.rand(*w.shape[:-1], device="cuda") * 2.0 ** -16 + 2.0 ** -18, torch.randn(n, device="cuda")


@pytest.mark.parametrize("m,k,n", [(1, 256, 70), (4, 1024, 130), (3, 70, 33), (20, 300, 64), (64, 512, 260), (700, 256, 1000), (2100, 4096, 512)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_bias", [False, True])
def test_product(m, k, n, dtype, with_bias):
    """A few rows quantized on the way in, a few, many."""
    from viola_amd import nn
    x, w, sw, bias = _operands(m, k, n, dtype)
    b = bias if with_bias else None
    y = nn.int8_linear(x, w, sw, b, dtype=F32)
    expected, bound = oi.forward(x, w, sw, b)
    fits = expected.abs() < 3e38
    assert fits.float().mean() > 0.9 and torch.isfinite(y[fits]).all()
    assert oi.within(torch.where(fits, y, 0.0), torch.where(fits, expected, 0.0), torch.where(fits, bound, 0.0))


def test_experts():
    from viola_amd import nn
    for rows in (24, 900):
        x, w, sw, _ = _operands(rows, 256, 96, BF16, 3)
        ends = [0, rows // 3, rows // 3 + 5, rows - 4]
        y = nn.int8_grouped_linear(x, w, sw, torch.tensor(ends, dtype=torch.int32, device="cuda"), dtype=F32)
        assert (y[ends[3]:] == 0).all()
        for g in range(3):
            part = slice(ends[g], ends[g + 1])
            expected, bound = oi.forward(x[part], w[g], sw[g])
            assert (expected.abs() < 3e38).all() and oi.within(y[part], expected, bound)
