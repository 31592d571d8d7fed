"""The operators around a block on tensors as they lie on the device: broadcast dimensions and gradients, rows cut out of wider ones, odd addresses; against the
64-bit formulas (oracle.norms, oracle.routing).

Tolerances, as for the same operators on contiguous tensors: 16-bit results are rounded once, by 2^-8 (BF16) or 2^-11 (FP16) of each value; in 32 bits a sum of n
terms is off by at most n 2^-24 of its terms' magnitudes, with chains of at most 64 and 44 additions: 2^-16 of the 2-norm, for sums over rows of the 2-norm of the
terms' magnitudes."""

import pytest
import torch

from oracle import norms, routing

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SUMS = 2.0 ** -16


def _close(name, actual, expected, measure=None):
    expected = expected.double().cpu()
    measure = expected if measure is None else measure.double().cpu()
    assert actual.shape == expected.shape, name
    off = (actual.detach().double().cpu() - expected).norm()
    bound = UNIT[actual.dtype] * expected.norm() + SUMS * measure.norm() + (2.0 ** -25 * expected.numel() ** 0.5 if actual.dtype == F16 else 0.0)
    assert off <= bound, (name, off.item(), bound.item())


def _leaf(t):
    """A leaf for gradients that lies where t does."""
    leaf = t.detach().requires_grad_()
    assert leaf.stride() == t.stride() and leaf.data_ptr() == t.data_ptr()
    return leaf


def _between(on, **options):
    """norm_between on device tensors as they are, forward and backward, against the formulas."""
    from viola_amd import nn
    torch.manual_seed(77)
    on = {k: _leaf(t) for k, t in on.items()}
    out, h = nn.norm_between(**on, **options)
    d_out, d_h = torch.randn(out.shape).to(out.dtype), torch.randn(h.shape).to(h.dtype)
    grads = torch.autograd.grad([out, h], list(on.values()), [d_out.cuda(), d_h.cuda()])
    expected = norms.norm(**{k: t.detach().cpu() for k, t in on.items()}, **options, dout=d_out, dh=d_h)
    _close("out", out, expected["out"])
    _close("h", h, expected["h"])
    for k, g in zip(on, grads):
        _close("d" + k, g, expected["d" + k], expected["m" + k] if k not in ("x", "y") else None)


def _vectors(b, c, dtype=F32):
    vector = lambda *shape: (0.3 * torch.randn(*shape) + 1).to(dtype).cuda()  # noqa: E731
    return dict(after_weight=vector(c), after_bias=vector(c), weight=vector(c), bias=vector(c), gate=vector(b, 1, c), scale=vector(b, 1, c), shift=vector(b, 1, c))


# ---------------------------------------------------------------------------------------------------------- broadcast dimensions
@pytest.mark.parametrize("c", [256, 250])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norms_of_broadcast_rows(c, dtype):
    """The residual stream or the block's result one row a sequence (strides c, 0, 1), one row for all, or one sequence for all."""
    torch.manual_seed(1)
    full = lambda: torch.randn(4, 9, c, device="cuda").to(dtype)  # noqa: E731
    row = torch.randn(4, 1, c, device="cuda").to(dtype).expand(4, 9, c)
    assert row.stride() == (c, 0, 1)
    for x, y in ((row, full()), (full(), row), (row, row), (torch.randn(c, device="cuda").to(dtype).expand(4, 9, c), full()),
                 (full(), torch.randn(1, 9, c, device="cuda").to(dtype).expand(4, 9, c))):
        _between(dict(x=x, y=y, **_vectors(4, c)), after="layer", before="rms")


@pytest.mark.parametrize("experts", [64, 30])
def test_router_of_broadcast_logits(experts):
    from viola_amd import nn
    torch.manual_seed(2)
    logits = _leaf(torch.randn(5, 1, experts, device="cuda").expand(5, 7, experts))
    assert logits.stride() == (experts, 0, 1)
    r = nn.route(logits, 3)
    there = logits.detach().cpu()
    chosen = routing.choose(there, 3)
    assert torch.equal(r.experts.cpu().long(), chosen) and torch.equal(r.positions.cpu().long(), routing.places(chosen, experts)[0])
    _close("gates", r.gates, routing.gates(there, chosen, "softmax", True, 1.0))
    dgates = torch.randn(5, 7, 3)
    grad, = torch.autograd.grad([r.gates, r.balance], logits, [dgates.cuda(), torch.tensor(1.5, device="cuda")])
    dense = _leaf(logits.detach().contiguous())
    again = nn.route(dense, 3)
    expected, = torch.autograd.grad([again.gates, again.balance], dense, [dgates.cuda(), torch.tensor(1.5, device="cuda")])
    assert torch.equal(grad, expected) and torch.equal(r.balance, again.balance)
    for a, b in zip(nn.balance_loss(logits, r.experts), nn.balance_loss(dense, r.experts)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cols", [256, 61])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_broadcast_tokens_and_gradients(cols, dtype):
    """Tokens that are one row a sequence on the way out, and the gradients of sums over tokens on the way back, which repeat each row."""
    from viola_amd import nn
    torch.manual_seed(3)
    b, s, k = 6, 10, 2
    chosen = routing.choose(torch.randn(b * s, 8), k, torch.rand(b * s) > 0.2)
    positions, counts, offsets = routing.places(chosen, 8)
    gates = torch.rand(b, s, k).cuda().requires_grad_()
    r = nn.Routing(positions.view(b, s, k).int().cuda(), offsets.int().cuda(), gates)
    x = _leaf(torch.randn(b, 1, cols, device="cuda").to(dtype).expand(b, s, cols))
    rows = nn.dispatch(x, r)
    assert torch.equal(rows.double().cpu(), routing.dispatch(x.detach().cpu().reshape(b * s, cols), positions, b * s * k))
    # the gradient of sums over ten places each: every row of it ten times
    d_rows = torch.randn(b * s * k // 10, cols).to(dtype)
    grad, = torch.autograd.grad(rows.view(-1, 10, cols).sum(1), x, d_rows.cuda())
    _close("dx", grad.view(b * s, cols), routing.combine(d_rows.repeat_interleave(10, 0), positions))
    y = torch.randn(b * s * k, cols).to(dtype)
    y_on = y.cuda().requires_grad_()
    seen = []
    out = nn.combine(y_on, r)
    out.register_hook(lambda g: seen.append(g.stride()))
    d = torch.randn(b, cols).to(dtype)
    dy, dg = torch.autograd.grad(out.sum(1), [y_on, gates], d.cuda())
    assert seen == [(cols, 0, 1)]
    expected, expected_gates = routing.combine_gradient(d.repeat_interleave(s, 0), y, positions, gates.detach().cpu().view(b * s, k))
    _close("dy", dy, expected)
    _close("dgates", dg.view(b * s, k), expected_gates, torch.full_like(expected_gates, cols ** 0.5))


# ---------------------------------------------------------------------------------------------------------- many groups
@pytest.mark.parametrize("with_weight", [False, True])
def test_vectors_for_more_than_two_million_tokens(with_weight):
    """More groups than one launch has slices for: a scale and a shift for each token. 64-bit formulas on the device; each gradient is one product, and the weight's a
    sum of 64 slices of 2^16 terms, whose partial sums and rounding errors both go as their root: 2^-24 2^8 of them, 2^-16 of the sum of all magnitudes."""
    from viola_amd import nn
    torch.manual_seed(5)
    n, c = (1 << 22) + 100, 8
    x, d = torch.randn(n, c, device="cuda"), torch.randn(n, c, device="cuda")
    scale, shift, weight = torch.randn(n, c, device="cuda"), torch.randn(n, c, device="cuda"), torch.rand(c, device="cuda")
    wanted = [t.requires_grad_() for t in ((scale, shift, weight) if with_weight else (scale, shift))]
    grads = torch.autograd.grad(nn.norm_before(x, weight, scale=scale, shift=shift), wanted, d)
    hat = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    expected = [d * hat * weight.detach(), d.double(), (d * hat * (1 + scale.detach())).sum(0)]
    measures = [expected[0], expected[1], (d * hat * (1 + scale.detach())).abs().sum(0)]
    for name, g, e, m in zip(("scale", "shift", "weight"), grads, expected, measures):
        assert (g.double() - e).norm() <= SUMS * m.norm(), name
