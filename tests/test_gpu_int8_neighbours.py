"""The 8-bit entry points write their results and nothing beside them, whatever the offsets hold: results are the middle of larger buffers of a pattern."""

import pytest
import torch

from oracle import int8 as oi

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: 0, BF16: 1, F16: 2}
BEFORE, BEHIND = 512, 1024                                                   # rows of pattern


class Middle:
    """rows x cols of `dtype` within rows of 0x5a"""

    def __init__(self, rows, cols, dtype):
        self.whole = torch.full((BEFORE + rows + BEHIND, cols * dtype.itemsize), 0x5a, dtype=torch.uint8, device="cuda")
        self.rows, self.dtype = rows, dtype
        self.t = self.whole[BEFORE:BEFORE + rows].view(dtype)

    def unharmed(self):
        return bool((self.whole[:BEFORE] == 0x5a).all() and (self.whole[BEFORE + self.rows:] == 0x5a).all())


def _call(name, *args):
    from viola_amd import _lib
    status = getattr(_lib.library(), name)(*(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return status


def _operands(m, n, k, groups=0):
    torch.manual_seed(m + n + k)
    pitch = -(-k // 16) * 16
    a = torch.zeros(m, pitch, dtype=torch.int8, device="cuda")
    a[:, :k] = torch.randint(-127, 128, (m, k), device="cuda")
    b = torch.randint(-127, 128, (max(groups, 1), n, pitch), dtype=torch.int8, device="cuda")
    return a, torch.rand(m, device="cuda"), b, torch.rand(max(groups, 1), n, device="cuda"), pitch


ODD_OFFSETS = [[0, 5, 3, 20], [-7, 4, 90, 12], [3, 8, 8, 9], [0, 1000, 1000, 2 ** 31 - 1], [50, 40, 30, -2 ** 31], [0, 2 ** 31 - 1, 0, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 300],
               [0, 700, 700, 700], [0, 0, 0, 0]]


@pytest.mark.parametrize("offsets", ODD_OFFSETS, ids=str)
@pytest.mark.parametrize("m,n,k", [(20, 40, 64), (48, 100, 70), (700, 130, 70), (700, 1030, 256), (2050, 264, 128)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_grouped_product(offsets, m, n, k, dtype):
    """Few rows, straight from registers, and tiles; rows in order and in range come out as their formula says."""
    a, sa, b, sb, pitch = _operands(m, n, k, 3)
    out, o = Middle(m, n, dtype), torch.tensor(offsets, dtype=torch.int32, device="cuda")
    assert _call("viola_int8_gemm", a, pitch, sa, b, pitch, n * pitch, sb, o, 3, m, n, k, None, 0, out.t, CODE[dtype]) == 0
    assert out.unharmed()
    if offsets == sorted(offsets) and offsets[0] == 0:
        ends = [min(v, m) for v in offsets]
        for g in range(3):
            rows = slice(ends[g], ends[g + 1])
            expected = (a[rows, :k].double() @ b[g, :, :k].double().t()) * sa[rows, None].double() * sb[g].double()
            assert oi.within(out.t[rows], expected, 3 * oi.U * expected.abs())
        assert (out.t[ends[3]:] == 0).all()


@pytest.mark.parametrize("offsets", [None] + ODD_OFFSETS, ids=str)
@pytest.mark.parametrize("m,n,k", [(700, 130, 70), (700, 1031, 256), (2050, 264, 128)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_gradient(offsets, m, n, k, dtype):
    a, sa, b, _, pitch = _operands(m, n, k, 3)
    z, dz = torch.randn(m, 2 * n, device="cuda").to(dtype), Middle(m, 2 * n, dtype)
    o = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    status = _call("viola_int8_gemm_gated_backward", a, pitch, sa, b, pitch, n * pitch, o, 0 if o is None else 3, m, n, k, z, 2 * n, CODE[dtype], 0, dz.t)
    assert status == 0 and dz.unharmed()
    if offsets is None:
        apart, dh = Middle(m, 2 * n, dtype), Middle(m, n, F32)
        assert _call("viola_int8_gemm", a, pitch, sa, b, pitch, 0, None, None, 0, m, n, k, None, 0, dh.t, 0) == 0
        assert _call("viola_int8_gated_backward", z, 2 * n, CODE[dtype], m, n, 0, dh.t, None, apart.t) == 0
        assert dh.unharmed() and apart.unharmed() and torch.equal(apart.t, dz.t)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 17), (70, 100), (33, 2049), (5, 8200), (19, 16400), (2100, 130)])
@pytest.mark.parametrize("offsets", [None] + ODD_OFFSETS[:7], ids=str)
@pytest.mark.parametrize("sums", [False, True])
def test_quantizer_with_factors(rows, cols, offsets, sums):
    from viola_amd import _lib
    torch.manual_seed(rows + cols)
    pitch, x = -(-cols // 16) * 16, torch.randn(rows, cols, device="cuda").to(BF16)
    factors = torch.rand(3 * cols + 4, device="cuda")
    parts = _lib.library().viola_int8_sum_parts(rows, cols)
    codes, scales, partial = Middle(rows, pitch, torch.int8), Middle(rows, 1, F32), Middle(parts, cols, F32)
    o = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    assert _call("viola_int8_quantize", x, cols, 1, rows, cols, -1, factors, o, 0 if o is None else 3, codes.t, pitch, scales.t, partial.t if sums else None) == 0
    assert codes.unharmed() and scales.unharmed() and partial.unharmed() and (codes.t[:, cols:] == 0).all()
    if sums:
        total, size = partial.t.double().sum(0), x.double().abs().sum(0)
        assert ((total - x.double().sum(0)).abs() <= rows * oi.U * size).all()
    else:
        assert (partial.whole == 0x5a).all()
    if o is None:
        v = x.double() * factors[:cols].double()
        q, s, loose, _ = oi.quantize(v, oi.U * v.abs())
        # the scale is of a product rounded once, and rounded itself
        assert ((scales.t.double() - s).abs() <= 3 * oi.U * s).all() and ((codes.t[:, :cols].double() - q).abs() <= loose.double()).all()


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 1000, 4096), (3, 33, 48), (4, 130, 2048)])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("activation", [-1, 0])
def test_few_rows_at_any_address_of_x(m, n, k, shift, activation):
    """x at any address and distance of its rows that its type allows; weights at no other than 16 bytes'."""
    torch.manual_seed(n)
    cols = k * (2 if activation >= 0 else 1)
    b, sb, out = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda"), torch.rand(n, device="cuda"), Middle(m, n, BF16)
    x = torch.randn(m, cols, device="cuda").to(BF16)
    store = torch.zeros(m * (cols + 3) + 8, device="cuda", dtype=BF16)
    placed = store[shift:shift + m * (cols + 3)].view(m, cols + 3)[:, :cols]
    placed.copy_(x)
    assert _call("viola_int8_rows_linear", placed, cols + 3, 1, m, k, activation, b, k, sb, n, None, 0, out.t, 1) == 0
    aligned = Middle(m, n, BF16)
    assert _call("viola_int8_rows_linear", x, cols, 1, m, k, activation, b, k, sb, n, None, 0, aligned.t, 1) == 0
    assert out.unharmed() and torch.equal(out.t, aligned.t)
    assert oi.within(out.t, *oi.forward(x, b, sb, None, None if activation < 0 else "silu"))
    assert _call("viola_int8_rows_linear", x, cols, 1, m, k, activation, b.data_ptr() + 8, k, sb, n, None, 0, out.t, 1) == -1
    assert _call("viola_int8_rows_linear", x, cols, 1, m, k, activation, b, k + 8, sb, n, None, 0, out.t, 1) == -1
