"""nn.quantize_int8, int8_linear, int8_grouped_linear and their modules against the 64-bit formulas (oracle.int8): sizes around the tiles, odd widths, types, strides, groups
that are empty, rows behind the last group, rows of zeros, of infinities and of tiny values, gradients, streams, and a run of a whole mixture of experts.

Tolerances are oracle.int8's bounds, value by value: codes are equal where no error lies behind them."""

import math

import pytest
import torch

from oracle import int8 as oi

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _weights(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-128, 128, shape, device="cuda", generator=g, dtype=torch.int8)
    return codes, torch.rand(shape[:-1], device="cuda", generator=g) * 0.01 + 1e-4


def _rows(rows, cols, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    return x.to(dtype)


SHAPES = [(1, 1, 1), (1, 16, 16), (2, 15, 31), (3, 17, 5), (8, 1024, 512), (16, 256, 96), (17, 48, 64), (33, 64, 40), (65, 320, 1), (127, 130, 129), (128, 128, 128), (129, 144, 257),
          (257, 1000, 300), (300, 770, 1000), (64, 2049, 70), (20, 8200, 40), (5, 16500, 33), (1000, 256, 2048), (2100, 512, 2304), (4000, 192, 4100), (700, 4096, 640)]


@pytest.mark.parametrize("cols", [1, 7, 8, 16, 130, 511, 512, 513, 1024, 2048, 2056, 4096, 8192, 8200, 16384, 16400, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_codes(cols, dtype):
    """Bit for bit: scales are 32-bit quotients, codes the nearest integers of exact quotients."""
    from viola_amd import nn
    x = _rows(37, cols, dtype)
    x[3] = 0
    x[5] *= 2.0 ** -14                                                       # subnormal in fp16
    codes, scale = nn.quantize_int8(x)
    q, s, _, _ = oi.quantize(x.double())
    assert codes.dtype == torch.int8 and scale.dtype == F32 and codes.shape == x.shape
    assert torch.equal(scale.double(), s[:, 0]) and torch.equal(codes.double(), q)


def test_codes_next_to_halves():
    """Quotients whose 32-bit value is a half while the exact one is not, and halves themselves, which go to the even integer."""
    from viola_amd import nn
    x = torch.zeros(4, 512, device="cuda")
    for row, amax in enumerate((127.0, 1.0, 3.0, 0.7)):
        s = torch.tensor(amax, device="cuda") / 127
        half = (torch.arange(126, device="cuda") + 0.5).double() * s.double()
        near = half.float()
        x[row, :126], x[row, 126:252] = near, torch.nextafter(near, torch.tensor(0.0, device="cuda"))
        x[row, 252:378], x[row, 378:504] = torch.nextafter(near, torch.tensor(math.inf, device="cuda")), -near
        x[row, 504] = amax
    codes, scale = nn.quantize_int8(x)
    q, s, _, _ = oi.quantize(x.double())
    assert torch.equal(scale.double(), s[:, 0]) and torch.equal(codes.double(), q)


@pytest.mark.parametrize("size", [2.0 ** -149, 2.0 ** -140, 2.0 ** -127, 2.0 ** -100, 2.0 ** -64, 2.0 ** -60, 2.0 ** 100, 3e38])
def test_codes_of_tiny_and_large_rows(size):
    from viola_amd import nn
    x = (_rows(9, 96, F32).clamp(-1, 1) * size)
    codes, scale = nn.quantize_int8(x)
    q, s, _, _ = oi.quantize(x.double())
    assert torch.equal(scale.double(), s[:, 0]) and torch.equal(codes.double(), q)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cols", [40, 2500, 20000])
def test_a_row_that_is_no_number(value, cols):
    from viola_amd import nn
    x = _rows(6, cols, BF16)
    x[2, cols // 2] = value
    codes, scale = nn.quantize_int8(x)
    assert torch.isnan(scale[2]) and (codes[2] == 0).all() and torch.isfinite(scale[[0, 1, 3, 4, 5]]).all()
    w, sw = _weights(24, cols)
    y = nn.int8_linear(x, w, sw)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4, 5]]).all()


def _check_linear(x, w, sw, bias=None, activation=None, dtype=None, weight_t=None):
    from viola_amd import nn
    x = x.detach().requires_grad_()
    b = None if bias is None else bias.detach().requires_grad_()
    y = nn.int8_linear(x, w, sw, b, activation=activation, dtype=dtype, weight_t=weight_t)
    flat = x.detach().reshape(-1, x.shape[-1])
    expected, bound = oi.forward(flat, w, sw, bias, activation)
    assert y.shape == (*x.shape[:-1], w.shape[0]) and y.dtype == (dtype or x.dtype)
    assert oi.within(y.reshape(expected.shape), expected, bound)
    dy = _rows(flat.shape[0], w.shape[0], y.dtype, seed=2).reshape(y.shape)
    wanted = [x] if b is None else [x, b]
    grads = torch.autograd.grad(y, wanted, dy)
    expected, bound = oi.backward(dy.reshape(-1, w.shape[0]), w, sw, flat, activation)
    assert grads[0].dtype == x.dtype and grads[0].shape == x.shape and oi.within(grads[0].reshape(expected.shape), expected, bound)
    if b is not None:                                                        # chains of at most 64 sums and 1024 rows of them
        d = dy.reshape(-1, w.shape[0]).double()
        assert grads[1].dtype == b.dtype and oi.within(grads[1], d.sum(0), 2048 * oi.U * d.abs().sum(0))
    return y, grads


@pytest.mark.parametrize("tokens,width,out", SHAPES)
def test_linear(tokens, width, out):
    w, sw = _weights(out, width)
    _check_linear(_rows(tokens, width, BF16), w, sw, _rows(1, out, F32, seed=5)[0])


@pytest.mark.parametrize("tokens,width,out", [(1, 8192, 40), (2, 4096, 65), (7, 2032, 33), (16, 512, 70), (16, 528, 70), (17, 1024, 130), (20, 1024, 9000), (32, 272, 8200), (48, 512, 700),
                                              (130, 1024, 520), (512, 128, 768), (512, 128, 769), (513, 128, 700), (300, 9008, 200), (260, 8208, 272), (3000, 128, 3000), (9000, 200, 4200), (9, 131072, 20)])
def test_ways_of_a_product(tokens, width, out):
    """Rows quantized on the way in, few rows, one to four tiles of channels a wavefront, tiles of each size, long sums: on the borders between them."""
    w, sw = _weights(out, width)
    _check_linear(_rows(tokens, width, BF16), w, sw * 0.1, _rows(1, out, F32, seed=5)[0])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
def test_few_rows_are_quantized_as_many(dtype, activation):
    """The same bits from one launch as from two, at any address of x."""
    from viola_amd import nn
    for tokens, width, out in ((1, 1024, 100), (3, 2560, 33), (2, 4096, 40), (4, 2032, 65), (8, 1024, 64), (15, 48, 17)):
        w, sw = _weights(out, width)
        store = _rows(600, 2 * width + 3, dtype).clamp(-30, 30)
        cols = width * (2 if activation else 1)
        for first in (0, 1, 3):
            many = nn.int8_linear(store[:, first:first + cols], w, sw, activation=activation)
            few = nn.int8_linear(store[:tokens, first:first + cols], w, sw, activation=activation)
            assert torch.equal(few, many[:tokens])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("result", [None, F32, BF16, F16])
@pytest.mark.parametrize("tokens,width,out", [(9, 200, 72), (260, 384, 136), (33, 100, 51)])
def test_types(dtype, result, tokens, width, out):
    w, sw = _weights(out, width)
    _check_linear(_rows(tokens, width, dtype).clamp(-4, 4), w, sw * 0.1, _rows(1, out, dtype, seed=5)[0], dtype=result)


@pytest.mark.parametrize("activation", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("tokens,width,out,dtype", [(1, 64, 48, BF16), (37, 129, 65, F16), (300, 1024, 520, BF16), (50, 2056, 40, F32), (3, 16400, 24, BF16), (700, 72, 2080, BF16), (700, 333, 65, F32)])
def test_gated(activation, tokens, width, out, dtype):
    w, sw = _weights(out, width)
    _check_linear(_rows(tokens, 2 * width, dtype).clamp(-30, 30), w, sw * 0.1, activation=activation)


@pytest.mark.parametrize("shape", [(2, 3, 64), (64,), (1, 1, 64), (0, 64), (3, 0, 64)])
def test_leading_dimensions(shape):
    w, sw = _weights(40, 64)
    _check_linear(_rows(max(1, math.prod(shape[:-1])), 64, BF16)[:math.prod(shape[:-1])].reshape(shape), w, sw, _rows(1, 40, BF16)[0])


def test_strided_operands():
    """Columns of a wider tensor, transposed rows, codes with a distance of their own, unaligned codes, transposed codes given and not."""
    from viola_amd import nn
    wide = _rows(70, 300, BF16)
    w, sw = _weights(96, 144)
    for x in (wide[:, 5:149], wide[:, 8:152], _rows(144, 70, BF16).t(), wide[::2, :144], wide[:1, :144].expand(70, 144)):
        _check_linear(x, w, sw)
    x = wide[:, :130]
    stored = torch.randint(-128, 128, (96, 160), device="cuda", dtype=torch.int8)
    flat = torch.randint(-128, 128, (96 * 130 + 5,), device="cuda", dtype=torch.int8)
    for w in (stored[:, :130], stored[:, 3:133], flat[5:].view(96, 130), torch.randint(-128, 128, (130, 96), device="cuda", dtype=torch.int8).t(), stored[:1, :130]):
        ours, _ = _check_linear(x, w, sw[:w.shape[0]])
        again, _ = _check_linear(x, w, sw[:w.shape[0]], weight_t=w.t())
        third, _ = _check_linear(x, w, sw[:w.shape[0]], weight_t=w.t().contiguous())
        assert torch.equal(ours, again) and torch.equal(ours, third)
    s2 = torch.stack([sw, sw], 1)[:, 0]
    assert torch.equal(nn.int8_linear(wide[:, :144], _weights(96, 144)[0], s2), nn.int8_linear(wide[:, :144], _weights(96, 144)[0], sw))


def test_longest_sums():
    """131072 products of the largest integers still fit their sum."""
    from viola_amd import nn
    x = torch.ones(3, 131072, device="cuda")
    w = torch.full((17, 131072), -128, device="cuda", dtype=torch.int8)
    y = nn.int8_linear(x, w, torch.ones(17, device="cuda"))
    expected = -128.0 * 127 * 131072 * (torch.ones((), device="cuda") / 127).double()
    assert ((y.double() - expected).abs() <= 4 * oi.U * expected.abs()).all()
    with pytest.raises(RuntimeError, match="at most 131072"):
        nn.int8_linear(torch.ones(3, 131073, device="cuda"), torch.zeros(2, 131073, device="cuda", dtype=torch.int8), torch.ones(2, device="cuda"))


GROUPS = [([5], 0), ([0, 0, 3], 0), ([0, 5, 0, 130, 1], 7), ([300, 0, 17, 128, 129, 256], 0), ([0, 0, 0], 20), ([1] * 70 + [0] * 30 + [33] * 31, 3), ([2, 1, 0, 4] * 16, 0),
          ([700, 20, 900, 0, 500], 200), ([16, 17, 15, 32], 1), ([20, 21, 0, 19] * 40, 30), ([1, 0] * 512, 0), ([3000, 1, 0, 2900], 900), ([33] * 65, 0)]


@pytest.mark.parametrize("counts,left", GROUPS)
@pytest.mark.parametrize("width,out,activation,dtype", [(128, 96, None, BF16), (70, 33, None, F32), (256, 272, "silu", BF16), (48, 40, "gelu", F16)])
def test_grouped(counts, left, width, out, activation, dtype):
    from viola_amd import nn
    groups, used = len(counts), sum(counts)
    w, sw = _weights(groups, out, width)
    sw = sw * 0.2
    x = _rows(used + left, width * (2 if activation else 1), dtype).clamp(-30, 30)
    x[used:] = math.nan                                                      # nobody's rows are not read into a result
    x.requires_grad_()
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    y = nn.int8_grouped_linear(x, w, sw, offsets, activation=activation)
    dy = _rows(used + left, out, y.dtype, seed=2)
    dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
    assert (y[used:] == 0).all() and (dx[used:] == 0).all()
    at = 0
    for e, n in enumerate(counts):
        if n:
            rows = x.detach()[at:at + n]
            assert oi.within(y[at:at + n], *oi.forward(rows, w[e], sw[e], None, activation)), e
            assert oi.within(dx[at:at + n], *oi.backward(dy[at:at + n], w[e], sw[e], rows, activation)), e
            alone = nn.int8_linear(rows, w[e], sw[e], activation=activation)
            assert torch.equal(alone, y[at:at + n]), e                       # sums are exact, whatever the tiles
        at += n
    turned = w.transpose(1, 2).contiguous()
    dx2, = torch.autograd.grad(nn.int8_grouped_linear(x, w, sw, offsets, activation=activation, weight_t=turned), x, dy)
    assert torch.equal(dx, dx2)


def test_grouped_strided_weights():
    """Every second expert of a larger store, and rows with a distance of their own."""
    from viola_amd import nn
    store, sw = _weights(8, 64, 160)
    w, s = store[::2, 4:52, :150], sw[::2, 4:52]
    x = _rows(50, 150, BF16)
    offsets = torch.tensor([0, 10, 10, 41, 50], dtype=torch.int32, device="cuda")
    y = nn.int8_grouped_linear(x, w, s, offsets)
    assert torch.equal(y, nn.int8_grouped_linear(x, w.contiguous(), s.contiguous(), offsets))
    assert oi.within(y[10:41], *oi.forward(x[10:41], w[2], s[2]))


@pytest.mark.parametrize("offsets", [[0, 5, 3, 20], [-7, 4, 90, 12], [3, 8, 8, 9], [0, 1000, 1000, 2 ** 31 - 1], [50, 40, 30, -2 ** 31]])
def test_offsets_out_of_order_stay_inside(offsets):
    """Values are undefined there; memory around the rows is not touched (the result is a part of a larger buffer's size, checked by its neighbours)."""
    from viola_amd import nn
    w, sw = _weights(3, 40, 64)
    x = _rows(20, 64, BF16).requires_grad_()
    guard = [torch.full((20, 40), 7.0, device="cuda", dtype=BF16) for _ in range(8)]
    y = nn.int8_grouped_linear(x, w, sw, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    y.backward(torch.ones_like(y))
    torch.cuda.synchronize()
    assert y.shape == (20, 40) and all((g == 7).all() for g in guard)


def test_gradient_beside_the_unrounded_layer():
    """The gradient of the layer without rounding, whose codes are at most half a step off: |dx - dy W| <= sum_n s' |w_n| / 2, through an activation times its slopes."""
    w, sw = _weights(80, 112)
    real = w.double() * sw.double()[:, None]
    for activation in (None, "silu", "gelu"):
        x = _rows(30, 112 * (2 if activation else 1), F32).clamp(-8, 8)
        _, (dx,) = _check_linear(x, w, sw, activation=activation)
        dy = _rows(30, 80, F32, seed=2)
        z = x.double()
        h = 1e-5
        # central differences of sum(dy * layer(z)), all rows at once as they do not meet
        def value(z):
            v = z if activation is None else oi.gate(z[:, :112], activation)[0] * z[:, 112:]
            return ((v @ real.t()) * dy.double()).sum(-1)
        differences = torch.stack([(value(z + h * e) - value(z - h * e)) / (2 * h) for e in torch.eye(z.shape[1], device="cuda", dtype=torch.float64)], -1)
        step = (dy.double() * sw.double()).abs().amax(-1, keepdim=True) / 127
        bound = (step / 2 * w.double().abs().sum(0) * (1 + 1e-5)).expand(30, 112)
        if activation:
            act, slope = oi.gate(z[:, :112], activation)
            bound = torch.cat([bound * (z[:, 112:] * slope).abs(), bound * act.abs()], -1)
        assert ((dx.double() - differences).abs() <= bound + 1e-5 * (1 + differences.abs())).all()


def test_wanted_gradients_alone():
    from viola_amd import nn
    w, sw = _weights(64, 96)
    x, bias = _rows(200, 96, BF16), _rows(1, 64, F32)[0]
    dy = _rows(200, 64, BF16, seed=2)
    both = torch.autograd.grad(nn.int8_linear(x.requires_grad_(), w, sw, bias.requires_grad_()), [x, bias], dy)
    only_x, = torch.autograd.grad(nn.int8_linear(x, w, sw, bias.detach()), x, dy)
    only_bias, = torch.autograd.grad(nn.int8_linear(x.detach(), w, sw, bias), bias, dy)
    assert torch.equal(both[0], only_x) and torch.equal(both[1], only_bias)
    y = nn.int8_linear(x, w, sw, bias)
    y.sum().backward()                                                       # a broadcast gradient
    assert oi.within(x.grad, *oi.backward(torch.ones(200, 64, device="cuda"), w, sw))
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = nn.int8_linear(x, w, sw, bias)
    with pytest.raises(NotImplementedError, match="once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    y = nn.int8_linear(x, w, sw, bias)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 1000), (5000, 70), (4100, 520), (2500, 2049), (1100, 4104), (40, 9000), (700, 16384), (33, 16400)])
def test_bias_gradient(rows, cols):
    """Sums over rows that one block, several and the longest rows' leave."""
    from viola_amd import nn
    w, sw = _weights(cols, 16)
    bias = torch.zeros(cols, device="cuda", requires_grad=True)
    dy = _rows(rows, cols, BF16, seed=3)
    nn.int8_linear(_rows(rows, 16, BF16), w, sw, bias).backward(dy)
    d = dy.double()
    assert oi.within(bias.grad, d.sum(0), 2048 * oi.U * d.abs().sum(0))


def test_another_stream_and_two_at_once():
    from viola_amd import nn
    w, sw = _weights(512, 1024)
    xs = [_rows(400, 1024, BF16, seed=s) for s in range(4)]
    expected = [nn.int8_linear(x, w, sw) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            results.append(nn.int8_linear(x, w, sw))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results, expected))


def test_replayed_forward():
    """Without a gradient: a captured forward pass of the grouped and the plain product, replayed with eager work in between, follows new inputs and offsets."""
    from viola_amd import nn
    w, sw = _weights(4, 64, 128)
    d, sd = _weights(48, 64)
    x = _rows(60, 128, BF16)
    offsets = torch.tensor([0, 10, 30, 30, 60], dtype=torch.int32, device="cuda")

    def step():
        with torch.no_grad():
            return nn.int8_linear(nn.int8_grouped_linear(x, w, sw, offsets), d, sd)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        x.copy_(_rows(60, 128, BF16, seed=replay + 10))
        offsets.copy_(torch.tensor([0, 3 * replay, 20, 45, 60 - replay], dtype=torch.int32))
        captured.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, step())


def test_refusals():
    from viola_amd import nn
    w, sw = _weights(24, 32)
    x = _rows(4, 32, BF16)
    e, se = _weights(3, 24, 32)
    offsets = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda")
    bad = [lambda: nn.int8_linear(x, w.float(), sw), lambda: nn.int8_linear(x, w, sw.double()), lambda: nn.int8_linear(x, w, sw[:5]), lambda: nn.int8_linear(x[:, :31], w, sw),
           lambda: nn.int8_linear(x, w, sw, torch.zeros(23, device="cuda")), lambda: nn.int8_linear(x, w, sw.requires_grad_()), lambda: nn.int8_linear(x.double(), w, sw),
           lambda: nn.int8_linear(x, e, se), lambda: nn.int8_linear(x, w, sw.detach(), weight_t=w), lambda: nn.int8_linear(x, w.cpu(), sw.detach()),
           lambda: nn.int8_linear(x, w, sw.detach(), dtype=torch.int8), lambda: nn.int8_linear(x, w, sw.detach(), activation="silu"),
           lambda: nn.int8_grouped_linear(x, torch.zeros(1025, 4, 32, dtype=torch.int8, device="cuda"), torch.zeros(1025, 4, device="cuda"),
                                          torch.zeros(1026, dtype=torch.int32, device="cuda")),
           lambda: nn.int8_grouped_linear(x, w, sw.detach(), offsets), lambda: nn.int8_grouped_linear(x, e, se, offsets.long()),
           lambda: nn.int8_grouped_linear(x, e, se, offsets[:3]), lambda: nn.int8_grouped_linear(x, e, se, offsets.cpu()), lambda: nn.int8_grouped_linear(x[None], e, se, offsets),
           lambda: nn.quantize_int8(x[:, :31], activation="silu"), lambda: nn.quantize_int8(x.long()), lambda: nn.quantize_int8(torch.zeros(3, 0, device="cuda"))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: nn.int8_linear(x, w, sw.detach(), activation="tanh"), lambda: nn.quantize_int8(x, activation="swish")):
        with pytest.raises(AssertionError):
            call()


def test_modules():
    import viola_amd
    from viola_amd import nn
    torch.manual_seed(3)
    source = torch.nn.Linear(100, 72, device="cuda", dtype=BF16)
    for cached in (False, True):
        layer = nn.Int8Linear.from_float(source, cache_transpose=cached)
        q, s, _, _ = oi.quantize(source.weight.detach().double())
        assert torch.equal(layer.weight.double(), q) and torch.equal(layer.weight_scale.double(), s[:, 0])
        x = _rows(30, 100, BF16).requires_grad_()
        y = layer(x)
        assert oi.within(y, *oi.forward(x.detach(), layer.weight, layer.weight_scale, layer.bias.detach()))
        y.backward(_rows(30, 72, BF16, seed=2))
        assert oi.within(x.grad, *oi.backward(_rows(30, 72, BF16, seed=2), layer.weight, layer.weight_scale)) and layer.bias.grad.dtype == BF16
        half = layer.half()
        assert half.weight_scale.dtype == F32 and half.weight.dtype == torch.int8 and half.bias.dtype == F16
        other = nn.Int8Linear(100, 72, cache_transpose=cached, device="cuda", dtype=F16)
        other.load_state_dict(half.state_dict())
        z = _rows(5, 100, F16).requires_grad_()
        assert torch.equal(other(z), half(z))
        assert torch.equal(torch.autograd.grad(other(z).sum(), z)[0], torch.autograd.grad(half(z).sum(), z)[0])
    fp8 = viola_amd.nn.Linear(64, 48, device="cuda", dtype=BF16)
    layer = nn.Int8Linear.from_float(fp8)
    assert (layer.dequantize_weight() - fp8.dequantize_weight().float()).abs().max() <= layer.weight_scale.max() * 0.5001
    experts = nn.GroupedExperts(4, 64, 96, device="cuda")
    ours = nn.Int8Experts.from_float(experts, activation="silu", cache_transpose=True)
    assert ours.weight.shape == (4, 96, 64) and ours.weight_t.shape == (4, 64, 96)
    y = ours(_rows(10, 128, BF16), torch.tensor([0, 4, 4, 8, 10], dtype=torch.int32, device="cuda"))
    assert y.shape == (10, 96)


@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_a_mixture_of_experts(tokens):
    """Router, dispatch, both products of the experts with the gate between them, combine: forward against the formulas step by step, and gradients that reach the logits and x."""
    from viola_amd import nn
    torch.manual_seed(tokens)
    experts, width, inner, top_k = 16, 96, 80, 4
    up, sup = _weights(experts, 2 * inner, width, seed=8)
    down, sdown = _weights(experts, width, inner, seed=9)
    x = _rows(tokens, width, BF16).requires_grad_()
    logits = torch.randn(tokens, experts, device="cuda", requires_grad=True)
    r = nn.route(logits, top_k)
    rows = nn.dispatch(x, r)
    z = nn.int8_grouped_linear(rows, up, sup * 0.05, r.offsets)
    out_rows = nn.int8_grouped_linear(z, down, sdown * 0.05, r.offsets, activation="silu")
    y = nn.combine(out_rows, r)
    bounds = r.offsets.tolist()
    for e in range(experts):
        a, b = bounds[e], bounds[e + 1]
        if a < b:
            assert oi.within(z[a:b], *oi.forward(rows.detach()[a:b], up[e], sup[e] * 0.05))
            assert oi.within(out_rows[a:b], *oi.forward(z.detach()[a:b], down[e], sdown[e] * 0.05, None, "silu"))
    dx, dl = torch.autograd.grad(y, [x, logits], _rows(tokens, width, BF16, seed=4))
    assert torch.isfinite(dx).all() and torch.isfinite(dl).all() and dx.abs().max() > 0 and (tokens == 1 or dl.abs().max() > 0)


@pytest.mark.parametrize("shape,width,inner", [((2, 61), 100, 72), ((3, 400), 128, 160), ((5, 1), 96, 40)])
def test_a_balanced_mixture_of_experts(shape, width, inner):
    """A router with a bias and groups over a padded batch, its rows through `Int8Experts`, and back: each step's forward and gradient against the formulas, on what the step was given."""
    from oracle import routing as ro
    from viola_amd import nn
    torch.manual_seed(shape[1])
    experts, top_k = 32, 6
    up = nn.Int8Experts.from_float(torch.randn(experts, 2 * inner, width, device="cuda") * 0.1, cache_transpose=True)
    down = nn.Int8Experts.from_float(torch.randn(experts, width, inner, device="cuda") * 0.1, activation="silu")
    tokens = shape[0] * shape[1]
    x = _rows(tokens, width, BF16).reshape(*shape, width).requires_grad_()
    logits = torch.randn(*shape, experts, device="cuda", requires_grad=True)
    bias = torch.randn(experts, device="cuda") * 0.1
    mask = torch.rand(shape, device="cuda") < 0.8
    mask[0, 0] = True
    r = nn.route(logits, top_k, score="sigmoid", bias=bias, groups=8, top_groups=4, group_top=2, mask=mask, per_sequence=True)
    chosen = ro.choose_steered(logits.detach().cpu(), top_k, "sigmoid", mask.cpu(), bias.cpu(), 8, 4, 2)
    assert torch.equal(r.experts.cpu().long(), chosen)
    rows = nn.dispatch(x, r)
    z = up(rows, r.offsets)
    out_rows = down(z, r.offsets)
    y = nn.combine(out_rows, r)
    dy = _rows(tokens, width, BF16, seed=4).reshape(*shape, width)
    d_rows, dz, d_out, dx, dl = torch.autograd.grad((y, r.balance), (rows, z, out_rows, x, logits), (dy, torch.ones((), device="cuda")))
    bounds = r.offsets.tolist()
    for e in range(experts):
        a, b = bounds[e], bounds[e + 1]
        if a < b:
            assert oi.within(z[a:b], *oi.forward(rows.detach()[a:b], up.weight[e], up.weight_scale[e]))
            assert oi.within(out_rows[a:b], *oi.forward(z.detach()[a:b], down.weight[e], down.weight_scale[e], None, "silu"))
            assert oi.within(dz[a:b], *oi.backward(d_out[a:b], down.weight[e], down.weight_scale[e], z.detach()[a:b], "silu"))
            assert oi.within(d_rows[a:b], *oi.backward(dz[a:b], up.weight[e], up.weight_scale[e]))
    for t in (z, out_rows, dz, d_rows):
        assert (t[bounds[-1]:] == 0).all()
    there = r.positions.cpu() >= 0
    gates, places = r.gates.detach().cpu().double() * there, r.positions.cpu().long().clamp(min=0)

    def sums(t, by):                                                         # top_k products and as many sums in 32 bits
        picked = t.detach().cpu().double()[places] * by[..., None]
        return picked.sum(-2), 2 * top_k * oi.U * picked.abs().sum(-2)

    assert oi.within(y.cpu(), *sums(out_rows, gates)) and oi.within(dx.cpu(), *sums(d_rows, there.double()))
    assert (y[~mask] == 0).all() and (dx[~mask] == 0).all() and (dl[~mask] == 0).all()
    # a gate's gradient is a dot product of `width` terms; what the logits' makes of its error is at most that error times the gate's slope, which is below one
    dots = (out_rows.detach().cpu().double()[places] * dy.cpu().double()[..., None, :])
    dgates, off = dots.sum(-1) * there, ((width + 1) * oi.U * dots.abs().sum(-1) * there).sum(-1, keepdim=True)
    expected = ro.gradient(logits.detach().cpu(), chosen, "sigmoid", mask.cpu(), True, dloss=1.0, dgates=dgates)
    spread = (dgates.abs().sum(-1, keepdim=True) + 1.0) * (4 * experts * oi.U)
    assert ((dl.cpu().double() - expected).abs() <= off + spread).all()


def test_a_served_mixture_is_replayed():
    """A decoding step of router, experts and combine in one graph: new tokens, a new bias and other places by each replay, with eager work in between."""
    from viola_amd import nn
    torch.manual_seed(7)
    experts, width, inner, tokens = 64, 128, 96, 12
    up = nn.Int8Experts.from_float(torch.randn(experts, 2 * inner, width, device="cuda") * 0.1)
    down = nn.Int8Experts.from_float(torch.randn(experts, width, inner, device="cuda") * 0.1, activation="silu")
    head = nn.Int8Linear.from_float(torch.nn.Linear(width, 70, device="cuda"))
    x, logits, bias = _rows(tokens, width, BF16), torch.randn(tokens, experts, device="cuda"), torch.zeros(experts, device="cuda")

    def step():                                                              # bias of `head` is a parameter: gradients are recorded, and only their pass has to be eager
        r = nn.route(logits, 8, score="sigmoid", bias=bias, groups=8, top_groups=3, group_top=2)
        return head(nn.combine(down(up(nn.dispatch(x, r), r.offsets), r.offsets), r)).detach(), r.experts

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        x.copy_(_rows(tokens, width, BF16, seed=replay + 20))
        logits.copy_(torch.randn(tokens, experts))
        bias.copy_(torch.randn(experts) * 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_a_captured_backward_pass_is_refused():
    """No eager graph of these leaves is alive, and the capture ends in order: refused by the nodes themselves before they launch anything."""
    from viola_amd import nn
    w, sw = _weights(48, 64)
    x, logits = _rows(20, 64, BF16).requires_grad_(), torch.randn(20, 16, device="cuda", requires_grad=True)
    bias = torch.zeros(16, device="cuda")
    dy, dg = _rows(20, 48, BF16, seed=2), torch.ones(20, 4, device="cuda")
    with torch.no_grad():
        nn.int8_linear(x, w, sw), nn.route(logits, 4, bias=bias)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        y, gates = nn.int8_linear(x, w, sw), nn.route(logits, 4, bias=bias).gates
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(y, x, dy)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(gates, logits, dg)
    torch.cuda.synchronize()
    dx, = torch.autograd.grad(nn.int8_linear(x, w, sw), x, dy)
    assert oi.within(dx, *oi.backward(dy, w, sw))


def test_more_rows_than_one_row_of_blocks():
    """2^26 and some rows of three values: more blocks of the quantizer than a grid has threads for in one dimension."""
    from viola_amd import nn
    rows = 2 ** 26 + 37
    x = torch.randn(rows, 3, device="cuda", dtype=BF16)
    w, sw = _weights(4, 3)
    codes, scale = nn.quantize_int8(x)
    y = nn.int8_linear(x, w, sw)
    for part in (slice(0, 1000), slice(2 ** 22 - 500, 2 ** 22 + 500), slice(2 ** 25, 2 ** 25 + 1000), slice(rows - 1000, rows)):
        q, s, _, _ = oi.quantize(x[part].double())
        assert torch.equal(scale[part].double(), s[:, 0]) and torch.equal(codes[part].double(), q)
        assert oi.within(y[part], *oi.forward(x[part], w, sw))


def test_codes_loaded_on_the_cpu_are_turned_on_the_way():
    from viola_amd import nn
    source = nn.Int8Linear.from_float(torch.nn.Linear(40, 24, device="cuda"), cache_transpose=True)
    layer = nn.Int8Linear(40, 24, cache_transpose=True)
    layer.load_state_dict({name: t.cpu() for name, t in source.state_dict().items()})
    assert layer.weight_t is None
    layer.cuda()
    assert torch.equal(layer.weight_t, source.weight_t)
    x = _rows(9, 40, F32)
    assert torch.equal(layer(x), source(x))
