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


# ---------------------------------------------------------------------------------------------------------- rows cut out of wider ones
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width,at_x,at_y,pieces", [(768, 0, 512, True), (768, 8, 264, True), (768, 257, 511, False), (768, 1, 512, False), (768, 0, 3, False), (771, 0, 0, False)])
def test_norms_of_rows_cut_out_of_wider_ones(dtype, width, at_x, at_y, pieces):
    """Rows of another distance than their width, from whole pieces of 16 bytes on or not, in a 3-D tensor whose rows still have one distance."""
    from viola_amd import _lib
    torch.manual_seed(6)
    wide = torch.randn(2, 4, 9, width, device="cuda").to(dtype)
    x, y = wide[0, ..., at_x:at_x + 256], wide[1, ..., at_y:at_y + 256]
    for t in (x, y):
        assert not t.is_contiguous() and _lib.host().row_layout(t) == (36, width, False)
    assert pieces == (x.data_ptr() % 16 == 0 and y.data_ptr() % 16 == 0 and width % 8 == 0)
    _between(dict(x=x, y=y, **_vectors(4, 256)), after="layer", before="rms")
    _between(dict(x=x, y=y, **_vectors(4, 256)), after="rms", before="layer")


def test_norms_of_rows_without_a_common_distance():
    torch.manual_seed(7)
    x, y = torch.randn(9, 4, 256, device="cuda").bfloat16().transpose(0, 1), torch.randn(4, 18, 256, device="cuda").bfloat16()[:, ::2]
    _between(dict(x=x, y=y, **_vectors(4, 256)))
    y = torch.randn(4, 12, 256, device="cuda").bfloat16()[:, :9]              # sequences further apart than their rows
    _between(dict(x=x, y=y, **_vectors(4, 256)))


def test_vectors_cut_out_of_wider_ones():
    """Gate, scale and shift as parts of one projection, aligned or not."""
    torch.manual_seed(8)
    for c, first in ((256, 0), (256, 3), (250, 1)):
        parts = (0.3 * torch.randn(4, 6 * 256 + 8, device="cuda")).bfloat16()
        cut = [parts[:, None, first + i * c:first + (i + 1) * c] for i in range(3)]
        x, y = torch.randn(4, 9, c, device="cuda").bfloat16(), torch.randn(4, 9, c, device="cuda").bfloat16()
        _between(dict(x=x, y=y, gate=cut[0], scale=cut[1], shift=cut[2]), after="rms", before="layer")


# ---------------------------------------------------------------------------------------------------------- many rows to a block
@pytest.mark.parametrize("c", [384, 1001, 1152, 4096])
@pytest.mark.parametrize("stream,branch", [(BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("options", [dict(after="rms", before="layer"), dict(after=None, before="rms")], ids=["normed", "plain"])
def test_blocks_of_many_rows(c, stream, branch, options):
    """Twelve to twenty rows to a block, in groups of 37 that begin and end inside one: teams of one to eight wavefronts make several turns, with the rows of the next ones
    under way and another group's vectors on the way."""
    torch.manual_seed(c)
    b, s = 136, 37
    given = dict(x=torch.randn(b, s, c, device="cuda").to(stream), y=torch.randn(b, s, c, device="cuda").to(branch))
    vectors = _vectors(b, c)
    if options["after"] is None:                                             # the kernel of its own: neither norm, weight nor bias after the block
        vectors = {k: v for k, v in vectors.items() if not k.startswith("after")}
    _between({**given, **vectors}, **options)


@pytest.mark.parametrize("form", ["before", "after"])
@pytest.mark.parametrize("c", [384, 1001, 1152])
def test_one_side_of_a_block_of_many_rows(form, c):
    from viola_amd import nn
    torch.manual_seed(c)
    b, s = 136, 37
    v = _vectors(b, c)
    if form == "before":
        on = dict(x=torch.randn(b, s, c, device="cuda"), weight=v["weight"], bias=v["bias"], scale=v["scale"], shift=v["shift"])
        call = lambda t: nn.norm_before(**t, kind="layer", dtype=BF16)  # noqa: E731
        options = dict(before="layer")
    else:
        on = dict(x=torch.randn(b, s, c, device="cuda"), y=torch.randn(b, s, c, device="cuda").bfloat16(), after_weight=v["after_weight"], after_bias=v["after_bias"], gate=v["gate"])
        call = lambda t: nn.norm_after(t["x"], t["y"], t["after_weight"], t["after_bias"], gate=t["gate"], kind="layer")  # noqa: E731
        options = dict(after="layer", before=None)
    on = {k: _leaf(t) for k, t in on.items()}
    result = call(on)
    d = torch.randn(b, s, c).to(result.dtype)
    grads = torch.autograd.grad(result, list(on.values()), d.cuda())
    expected = norms.norm(**{k: t.detach().cpu() for k, t in on.items()}, **options, **{"dh" if form == "before" else "dout": d})
    _close(form, result, expected["h" if form == "before" else "out"])
    for k, g in zip(on, grads):
        _close("d" + k, g, expected["d" + k], expected["m" + k] if k not in ("x", "y") else None)


def test_more_rows_than_the_caches_hold():
    """Inputs beyond 128 MB are read past the caches' order."""
    torch.manual_seed(9)
    x, y = torch.randn(8, 1026, 4096, device="cuda").bfloat16(), torch.randn(8, 1026, 4096, device="cuda").bfloat16()
    assert 2 * x.numel() * x.element_size() > 128 << 20
    _between(dict(x=x, y=y, **{k: v for k, v in _vectors(8, 4096).items() if k in ("after_weight", "weight", "gate")}))


@pytest.mark.parametrize("top_k", [1, 8])
def test_more_rows_of_experts_than_the_caches_hold(top_k):
    """The same on the way to the experts and back; a sample of the tokens against the formulas, every row against the rows of its token."""
    from viola_amd import nn
    torch.manual_seed(10)
    cols = 4096
    tokens = (128 << 20) // (2 * cols * top_k) + 5
    chosen = torch.randint(0, 16, (tokens, top_k))
    flat = chosen.flatten()
    positions = torch.empty_like(flat)
    positions[torch.argsort(flat, stable=True)] = torch.arange(flat.numel())
    positions = positions.view(tokens, top_k)
    offsets = torch.nn.functional.pad(torch.bincount(flat, minlength=16).cumsum(0), (1, 0))
    gates = torch.rand(tokens, top_k).cuda().requires_grad_()
    r = nn.Routing(positions.int().cuda(), offsets.int().cuda(), gates)
    x = torch.randn(tokens, cols, device="cuda").bfloat16()
    rows = nn.dispatch(x, r)
    assert torch.equal(rows[positions.cuda()], x[:, None].expand(-1, top_k, -1))
    y = torch.randn(tokens * top_k, cols, device="cuda").bfloat16().requires_grad_()
    d = torch.randn(tokens, cols, device="cuda").bfloat16()
    out = nn.combine(y, r)
    dy, dg = torch.autograd.grad(out, [y, gates], d)
    some = torch.randperm(tokens)[:200]
    at = positions[some].cuda()
    y64, d64, g64 = y.detach()[at].double(), d[some.cuda()].double(), gates.detach()[some.cuda()].double()
    _close("out", out[some.cuda()], (g64[..., None] * y64).sum(1))
    _close("dy", dy[at], g64[..., None] * d64[:, None])
    dots = (d64[:, None] * y64).sum(-1)
    _close("dgates", dg[some.cuda()], dots, torch.full_like(dots, cols ** 0.5))
