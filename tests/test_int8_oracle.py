"""oracle.int8 against brute force and differences, and what the operators of 8-bit integers refuse without a GPU."""

import pytest
import torch

from oracle import int8 as oi


def test_codes_by_brute_force():
    """The nearest of all 255 codes, a half to the even one."""
    torch.manual_seed(0)
    x = torch.randn(6, 40, dtype=torch.float64)
    x[1] = 0
    x[2, :5] = torch.tensor([0.5, 1.5, 2.5, -0.5, -3.5]) * (2.0 ** -3)
    x[2, 5], x[2, 6:] = 127 * 2.0 ** -3, 0.0
    codes, scale, loose, _ = oi.quantize(x)
    assert not loose.any() and (scale[1] == 0).all() and (codes[1] == 0).all()
    assert codes[2, :6].tolist() == [0, 2, 2, 0, -4, 127]
    levels = torch.arange(-127, 128, dtype=torch.float64)
    for r in (0, 3, 4, 5):
        nearest = levels[(x[r][:, None] - levels * scale[r]).abs().argmin(-1)]
        assert torch.equal(codes[r], nearest)


@pytest.mark.parametrize("activation", ["silu", "gelu", "relu"])
def test_slopes_by_differences(activation):
    g = torch.linspace(-12, 12, 241, dtype=torch.float64) + 0.013
    act, slope = oi.gate(g, activation)
    h = 1e-6
    assert torch.allclose((oi.gate(g + h, activation)[0] - oi.gate(g - h, activation)[0]) / (2 * h), slope, atol=1e-8)
    plain = dict(silu=torch.nn.functional.silu, relu=torch.relu, gelu=lambda v: torch.nn.functional.gelu(v, approximate="tanh"))[activation]
    assert torch.allclose(act, plain(g), atol=1e-12)
    # the bounds hold for the formula evaluated in 32 bits (torch's sigmoid is within 4 ulp of its own)
    f = g.float()
    a = f if activation == "silu" else f * (1.5957691216057308 + 0.0713548162726 * f * f)
    in32 = torch.relu(f) if activation == "relu" else f * torch.sigmoid(a)
    exact, _, off, _ = oi.gate(f.double(), activation, True)
    assert ((in32.double() - exact).abs() <= 2 * off).all()


def test_product_by_hand():
    x = torch.tensor([[127.0, -64.0, 0.4]])
    w = torch.tensor([[1, 2, 3], [-128, 0, 127]], dtype=torch.int8)
    y, bound = oi.forward(x, w, torch.tensor([0.5, 2.0]), torch.tensor([1.0, -1.0]))
    assert y.tolist() == [[(127 - 128) * 0.5 + 1, -128 * 127 * 2 - 1]] and (bound < 1e-2).all()
    dy = torch.tensor([[2.0, 127.0 / 2]])
    dx, _ = oi.backward(dy, w, torch.tensor([0.5, 2.0]))
    assert dx.tolist() == [[1 - 128 * 127, 2.0, 3 + 127 * 127]]


@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
def test_gradient_beside_the_unrounded_layer(activation):
    """Half a step of each code of the gradient, times the weights it meets."""
    torch.manual_seed(1)
    w, sw = torch.randint(-128, 128, (30, 20), dtype=torch.int8), torch.rand(30) * 0.01
    x = torch.randn(7, 20 * (2 if activation else 1), dtype=torch.float64).requires_grad_()
    dy = torch.randn(7, 30)
    v = x if activation is None else oi.gate(x[:, :20], activation)[0] * x[:, 20:]
    exact, = torch.autograd.grad(v @ (w.double() * sw.double()[:, None]).t(), x, dy.double())
    dx, _ = oi.backward(dy, w, sw, x.detach(), activation)
    bound = ((dy.double() * sw.double()).abs().amax(-1, keepdim=True) / 127 / 2 * w.double().abs().sum(0) * (1 + 1e-6)).expand(7, 20)
    if activation:
        act, slope = oi.gate(x.detach()[:, :20], activation)
        bound = torch.cat([bound * (x.detach()[:, 20:] * slope).abs(), bound * act.abs()], -1)
    assert ((dx - exact).abs() <= bound + 1e-12).all() and (dx != exact).any()


def _calls():
    from viola_amd import nn
    w, s = torch.zeros(6, 8, dtype=torch.int8), torch.zeros(6)
    places = torch.zeros(3, dtype=torch.int32)
    return {"quantize_int8": lambda t: nn.quantize_int8(t)[1], "int8_linear": lambda t: nn.int8_linear(t, w, s),
            "int8_grouped_linear": lambda t: nn.int8_grouped_linear(t, torch.zeros(2, 6, 8, dtype=torch.int8), torch.zeros(2, 6), places)}


@pytest.mark.parametrize("name", ["quantize_int8", "int8_linear", "int8_grouped_linear"])
def test_recorded_graphs_and_transforms_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = _calls()[name], torch.randn(4, 8)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="recorded"):
        torch.jit.trace(f, (x,), check_trace=False)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        make_fx(f)(x)
    with pytest.raises(NotImplementedError):
        torch.func.grad(lambda t: f(t).float().sum())(x)
    with pytest.raises(RuntimeError, match="GPU"):
        f(x)


def test_rejected_calls_launch_nothing():
    """Argument checks come before any launch; the pointers are never dereferenced."""
    from viola_amd import _lib
    lib = _lib.library()
    P, F32, BF16, E4M3 = 0x10000, 0, 1, 3
    q = lambda **c: lib.viola_int8_quantize(*{**dict(x=P, pitch=64, dtype=BF16, rows=4, cols=64, act=-1, factors=None, offsets=None, groups=0, codes=P, cp=64, scales=P,  # noqa: E731
                                                     partial=None), **c}.values(), None)
    for bad in (dict(dtype=E4M3), dict(rows=-1), dict(cols=0), dict(pitch=63), dict(act=3), dict(cp=48), dict(cp=72), dict(cp=96), dict(codes=P + 8), dict(scales=None), dict(x=None),
                dict(act=0), dict(factors=P, act=0, pitch=128), dict(offsets=P), dict(partial=P), dict(factors=P + 4), dict(factors=P, offsets=P)):
        assert q(**bad) == -1, bad
    assert q(rows=0) == 0
    g = lambda **c: lib.viola_int8_gemm(*{**dict(a=P, lda=64, sa=P, b=P, ldb=64, bs=0, sb=P, offsets=None, groups=0, m=4, n=8, k=64, bias=None, bt=F32, out=P, ot=BF16), **c}.values(),  # noqa: E731
                                        None)
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(ot=E4M3), dict(bias=P, bt=E4M3), dict(lda=48), dict(lda=72), dict(ldb=63), dict(a=P + 1), dict(b=P + 8), dict(out=None), dict(sa=None),
                dict(offsets=P), dict(offsets=P, groups=2, bias=P), dict(bs=8), dict(groups=-1), dict(m=1 << 31)):
        assert g(**bad) == -1, bad
    assert g(k=(1 << 17) + 1) == -2 and g(ldb=(1 << 22) + 16) == -2 and g(m=0) == 0
    assert g(m=(1 << 31) - 1, n=1 << 20) == -3                               # more tiles than a grid has threads for
    gb = lambda **c: lib.viola_int8_gemm_gated_backward(*{**dict(a=P, lda=64, sa=P, b=P, ldb=64, bs=0, offsets=None, groups=0, m=1000, n=800, k=64, z=P, zp=1600, zt=BF16, act=0,  # noqa: E731
                                                                 dz=P), **c}.values(), None)
    for bad in (dict(act=-1), dict(act=3), dict(zp=1599), dict(n=0), dict(zt=E4M3), dict(z=None), dict(dz=None), dict(lda=48), dict(m=-1), dict(offsets=P), dict(a=P + 4)):
        assert gb(**bad) == -1, bad
    assert gb(m=0) == 0 and gb(m=8) == -2 and gb(k=2064, lda=2064, ldb=2064) == -2
    r = lambda **c: lib.viola_int8_rows_linear(*{**dict(x=P, pitch=64, dtype=BF16, m=4, k=64, act=-1, b=P, ldb=64, sb=P, n=8, bias=None, bt=F32, out=P, ot=BF16), **c}.values(), None)  # noqa: E731
    for bad in (dict(dtype=E4M3), dict(pitch=63), dict(act=0), dict(act=3), dict(ldb=48), dict(ldb=72), dict(n=0), dict(sb=None), dict(b=P + 8), dict(out=None), dict(bias=P, bt=E4M3)):
        assert r(**bad) == -1, bad
    assert r(m=0) == 0 and r(m=17) == -2 and r(m=5) == -2 and r(k=40) == -2 and r(m=8, k=4096, pitch=4096, ldb=4096) == -2
    b = lambda **c: lib.viola_int8_gated_backward(*{**dict(z=P, pitch=64, dtype=BF16, rows=4, cols=32, act=0, dh=P, total=None, dz=P), **c}.values(), None)  # noqa: E731
    for bad in (dict(dtype=E4M3), dict(pitch=63), dict(act=-1), dict(act=3), dict(dh=None), dict(dz=None), dict(rows=-1)):
        assert b(**bad) == -1, bad
    assert b(rows=0) == 0 and lib.viola_int8_sum_parts(0, 5) == 0 and lib.viola_int8_sum_parts(7, 0) == 0


def test_sums_have_a_row_for_each_part():
    from viola_amd import _lib
    for rows in (1, 4, 5, 1000, 1025, 5000, 40000):
        for cols in (1, 512, 2049, 8192, 16384, 16385):
            parts = _lib.library().viola_int8_sum_parts(rows, cols)
            assert 0 < parts <= max(4096, (rows + 15) // 16), (rows, cols, parts)
