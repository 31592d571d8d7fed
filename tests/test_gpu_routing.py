"""nn.route / balance_loss / dispatch / combine against the 64-bit formulas (oracle.routing): counts of experts and choices, ties, masked tokens and experts, sequences, types,
strides, and the way of rows there and back.

Tolerances. In 32 bits a sum of n terms is off by at most n 2^-24 of the sum of their magnitudes, and an exponential by 2^-22; the longest chain here is 64 terms and
44 for joining: 2^-16 of the 2-norm, for the logits' gradient (a difference of two sums) of the 2-norm of its terms. 16-bit results are rounded once, by 2^-8 or 2^-11."""

import math

import pytest
import torch

from oracle import routing

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


def _pull(logits, chosen, score, mask, per_sequence, dloss, dgates, normalize, scale):
    """Magnitudes of the terms that the logits' gradient is the difference of."""
    p, _, _ = routing.probabilities(logits, score)
    p = p.nan_to_num()
    _, _, cost = routing.balance(logits, chosen, score, mask, per_sequence)
    cost = cost.repeat_interleave(math.prod(logits.shape[:-1]) // cost.shape[0], 0).reshape(p.shape)
    g = 0.0
    if dgates is not None:
        gates = routing.gates(logits, chosen, score, normalize, scale).abs()
        there = (chosen >= 0).double()
        part = torch.zeros(*p.shape[:-1], p.shape[-1] + 1, dtype=torch.float64)
        along = (gates * dgates.double().cpu().abs() * there).sum(-1, keepdim=True)
        part.scatter_add_(-1, torch.where(chosen >= 0, chosen, p.shape[-1]), gates * dgates.double().cpu().abs() * there + gates * along)
        g = part[..., :-1] + p * along
    return abs(dloss) * p * (cost + (p * cost).sum(-1, keepdim=True)) + g


def _check_route(logits, top_k, *, mask=None, score="softmax", normalize=True, scale=1.0, per_sequence=False, on=None):
    from viola_amd import nn
    torch.manual_seed(3)
    l = (logits.cuda() if on is None else on).detach().requires_grad_()
    r = nn.route(l, top_k, score=score, normalize=normalize, scale=scale, mask=None if mask is None else mask.cuda(), per_sequence=per_sequence)
    counted = routing.counted_tokens(logits, mask)
    chosen = routing.choose(logits, top_k, counted)
    positions, counts, offsets = routing.places(chosen, logits.shape[-1])
    for name, t, e in (("experts", r.experts, chosen), ("positions", r.positions, positions), ("counts", r.counts, counts), ("offsets", r.offsets, offsets)):
        assert t.dtype == torch.int32 and torch.equal(t.cpu().long(), e), name
    _close("gates", r.gates, routing.gates(logits, chosen, score, normalize, scale))
    loss, _, _ = routing.balance(logits, chosen, score, mask, per_sequence)
    _close("balance", r.balance, loss)
    dgates, dloss = torch.randn(r.gates.shape), 1.5
    for use in ((True, True), (True, False), (False, True)):
        outputs = [t for t, u in zip((r.gates, r.balance), use) if u]
        given = [t for t, u in zip((dgates.cuda(), torch.tensor(dloss, device="cuda")), use) if u]
        grad, = torch.autograd.grad(outputs, l, given, retain_graph=True)
        assert grad.dtype == l.dtype
        dl, dg = dloss * use[1], dgates if use[0] else None
        expected = routing.gradient(logits, chosen, score, mask, per_sequence, dloss=dl, dgates=dg, normalize=normalize, scale=scale)
        _close("dlogits", grad, expected, _pull(logits, chosen, score, mask, per_sequence, dl, dg, normalize, scale))
        assert (grad[~counted.cuda()] == 0).all()
    # the same choices handed to the loss alone
    for wide in (torch.int32, torch.int64):
        l2 = l.detach().requires_grad_()
        again, again_counts = nn.balance_loss(l2, r.experts.to(wide), score=score, mask=None if mask is None else mask.cuda(), per_sequence=per_sequence)
        assert torch.equal(again_counts.cpu().long(), counts)
        _close("balance", again, loss)
        grad, = torch.autograd.grad(again, l2)
        _close("dlogits", grad, routing.gradient(logits, chosen, score, mask, per_sequence, dloss=1.0),
               _pull(logits, chosen, score, mask, per_sequence, 1.0, None, True, 1.0))
    return r


@pytest.mark.parametrize("experts", [1, 2, 3, 8, 9, 16, 31, 32, 60, 64, 100, 128, 160, 256, 257, 384, 512, 700, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_experts(experts, score):
    torch.manual_seed(experts)
    _check_route(torch.randn(70, experts) * 2, min(experts, 4), score=score)


@pytest.mark.parametrize("top_k", [1, 2, 3, 5, 8, 13, 32])
@pytest.mark.parametrize("score,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_choices(top_k, score, normalize):
    torch.manual_seed(top_k)
    _check_route(torch.randn(90, 64), top_k, score=score, normalize=normalize, scale=2.5)


@pytest.mark.parametrize("shape", [(1, 64), (2, 64), (31, 8), (257, 8), (300, 3), (32, 64), (33, 64), (1000, 16), (4099, 12), (2, 2, 64), (3, 129, 64), (16, 77, 8), (300, 2, 4), (600, 1, 5), (3, 4, 5, 64)])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_tokens_and_sequences(shape, per_sequence):
    torch.manual_seed(shape[0])
    _check_route(torch.randn(shape), min(2, shape[-1]), per_sequence=per_sequence)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("experts", [16, 60, 63])
def test_types_and_ties(dtype, experts):
    """Logits on a coarse grid: most rows have ties, which go to the lowest index."""
    torch.manual_seed(4)
    _check_route((torch.randn(200, experts) * 2).round().div(2).to(dtype), 6)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_an_only_choice_has_no_gradient_from_its_gate(score):
    """Its share of itself is one whatever its logit: the balance loss's gradient is all there is, however small beside the gate's."""
    from viola_amd import nn
    torch.manual_seed(12)
    logits = torch.randn(300, 16)
    logits[:100, 1:] = -math.inf                                             # one open expert of two choices
    for part, top_k in ((logits[:100], 2), (logits[100:], 1)):
        l = part.cuda().requires_grad_()
        r = nn.route(l, top_k, score=score)
        grad, = torch.autograd.grad(r.gates, l, torch.randn(r.gates.shape, device="cuda"), retain_graph=True)
        assert (grad == 0).all()
        both, = torch.autograd.grad([r.gates, r.balance], l, [torch.randn(r.gates.shape, device="cuda"), torch.tensor(1e-6, device="cuda")])
        chosen = routing.choose(part, top_k)
        _close("dlogits", both, routing.gradient(part, chosen, score, dloss=1e-6), _pull(part, chosen, score, None, False, 1e-6, None, True, 1.0))


def test_all_equal_and_signed_zeros():
    logits = torch.zeros(40, 24)
    logits[::2, ::3] = -0.0
    r = _check_route(logits, 3)
    assert (r.experts.cpu() == torch.arange(3)).all()


@pytest.mark.parametrize("per_sequence", [False, True])
@pytest.mark.parametrize("score,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_masks(per_sequence, score, normalize):
    """Tokens left out (a whole sequence among them, with NaN and infinities inside), experts closed for some or all tokens."""
    torch.manual_seed(5)
    logits = torch.randn(6, 50, 32)
    mask = torch.rand(6, 50) < 0.7
    mask[2] = False
    logits[:, :, 7] = -math.inf                                              # closed for all
    logits[0, :10, 3:] = -math.inf                                           # fewer open than chosen
    logits[1, 4] = -math.inf                                                 # none open
    mask[1, 4] = mask[0, :10] = True
    clean = logits.clone()
    logits[2], logits[3][~mask[3]] = math.nan, math.inf                      # what a masked token holds must not matter
    clean[2], clean[3][~mask[3]] = 0.0, 0.0
    _check_route(clean, 4, mask=mask, score=score, normalize=normalize, per_sequence=per_sequence, on=logits.cuda())


def test_lowest_values_of_the_type():
    """Masks made of the type's lowest finite value can be chosen last, and count as experts with probability zero."""
    for dtype in (F32, BF16, F16):
        logits = torch.randn(20, 8).to(dtype)
        logits[:, 4:] = torch.finfo(dtype).min
        logits[3] = torch.finfo(dtype).min
        _check_route(logits, 6)
        _check_route(logits, 6, score="sigmoid")
        _check_route(logits, 2, normalize=False)


def test_far_from_zero():
    torch.manual_seed(6)
    for shift in (-300.0, -90.0, 90.0, 300.0):
        _check_route(torch.randn(50, 16) * 3 + shift, 3, score="sigmoid")
        _check_route(torch.randn(50, 16) * 3 + shift, 3, score="softmax")


def test_nan_and_infinity_in_counted_rows():
    """NaN is above all numbers and spreads over its own row only; choices stay in range."""
    from viola_amd import nn
    torch.manual_seed(7)
    logits = torch.randn(50, 16)
    logits[3, 5], logits[8, 2], logits[9] = math.nan, math.inf, math.nan
    l = logits.cuda().requires_grad_()
    r = nn.route(l, 4)
    chosen = routing.choose(logits, 4)
    assert torch.equal(r.experts.cpu().long(), chosen) and chosen[3, 0] == 5 and chosen[8, 0] == 2 and chosen[9].tolist() == [0, 1, 2, 3]
    assert torch.equal(r.positions.cpu().long(), routing.places(chosen, 16)[0])
    grad, = torch.autograd.grad(r.gates.sum() * 2 + (r.gates * r.gates).sum(), l)
    others = [i for i in range(50) if i not in (3, 8, 9)]
    assert r.gates[[3, 8, 9]].isnan().any(-1).all() and r.gates[others].isfinite().all()
    assert grad[[3, 8, 9]].isnan().any(-1).all() and grad[others].isfinite().all() and r.balance.isnan()


def test_strided_logits():
    torch.manual_seed(8)
    for shape, cut in (((40, 96), (slice(None), slice(32, 96))), ((40, 97), (slice(None), slice(33, 97))), ((40, 64, 2), (slice(None), slice(None), 1)), ((4, 10, 64), (slice(None), slice(2, 9)))):
        wide = torch.randn(shape)
        _check_route(wide[cut], 3, on=wide.cuda()[cut])
    _check_route(torch.randn(64, 30).t(), 3)
    row = torch.randn(1, 16)
    _check_route(row.expand(12, 16), 3, on=row.cuda().expand(12, 16))


def test_indices_out_of_range_count_nowhere():
    from viola_amd import nn
    torch.manual_seed(9)
    logits, chosen = torch.randn(100, 8), torch.randint(-3, 12, (100, 3))
    chosen[:, 1] = chosen[:, 0]                                              # the same one twice counts twice
    loss, counts = nn.balance_loss(logits.cuda(), chosen.cuda())
    inside = torch.where((chosen >= 0) & (chosen < 8), chosen, -1)
    expected, expected_counts, _ = routing.balance(logits, inside, "softmax")
    assert torch.equal(counts.cpu().double(), expected_counts)
    _close("balance", loss, expected)


def test_more_tokens_than_blocks_take_at_once():
    """Many passes of every block, by sums that are known: experts chosen in turn."""
    from viola_amd import nn
    tokens, experts = 100003, 64
    at = torch.arange(tokens, device="cuda")
    logits = torch.zeros(tokens, experts, device="cuda")
    logits[at, at % experts] = 4.0
    logits[at, (at * 7 + 3) % experts] += 2.0
    r = nn.route(logits, 2)
    flat = r.experts.flatten().long()
    assert torch.equal(r.counts.long(), torch.bincount(flat, minlength=experts))
    order = torch.argsort(flat, stable=True)
    expected = torch.empty_like(flat)
    expected[order] = torch.arange(flat.numel(), device="cuda")
    assert torch.equal(r.positions.flatten().long(), expected)
    p = torch.softmax(logits.double(), -1).mean(0)
    _close("balance", r.balance, experts * (r.counts.double() / (2 * tokens) * p).sum())


def test_no_tokens():
    from viola_amd import nn
    logits = torch.randn(2, 0, 8, device="cuda", requires_grad=True)
    r = nn.route(logits, 2)
    assert r.gates.shape == (2, 0, 2) and r.counts.tolist() == [0] * 8 and r.offsets.tolist() == [0] * 9 and r.balance == 0
    grad, = torch.autograd.grad(r.gates.sum() + r.balance, logits)
    assert grad.shape == logits.shape
    rows = nn.dispatch(torch.randn(2, 0, 16, device="cuda"), r)
    assert rows.shape == (0, 16) and nn.combine(rows, r).shape == (2, 0, 16)
    assert (nn.dispatch(torch.randn(2, 0, 16, device="cuda"), r, 3) == 0).all()


def test_routing_does_not_change_from_call_to_call():
    from viola_amd import nn
    torch.manual_seed(10)
    logits = torch.randn(16, 1000, 64, device="cuda", requires_grad=True)
    def call():
        r = nn.route(logits, 6, per_sequence=True)
        return (*r, *torch.autograd.grad(r.gates.square().sum() + r.balance, logits))
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))


# ---------------------------------------------------------------------------------------------------------- rows
def _places(tokens, experts, top_k, masked=0.0, seed=0):
    torch.manual_seed(seed)
    chosen = routing.choose(torch.randn(tokens, experts), top_k, torch.rand(tokens) >= masked)
    return routing.places(chosen, experts)


def _routing(positions, offsets, gates=None):
    from viola_amd import nn
    return nn.Routing(positions.int().cuda(), offsets.int().cuda(), None if gates is None else gates.cuda())


@pytest.mark.parametrize("cols", [1, 3, 8, 63, 64, 200, 512, 1000, 1024, 1152, 4096, 5001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_there_and_back(cols, dtype):
    from viola_amd import nn
    positions, counts, offsets = _places(37, 6, 2, masked=0.2, seed=cols)
    x, y, gates = torch.randn(37, cols).to(dtype), torch.randn(74, cols).to(dtype), torch.rand(37, 2)
    r = _routing(positions, offsets, gates.requires_grad_())
    on = x.cuda().requires_grad_()
    rows = nn.dispatch(on, r)
    assert rows.dtype == dtype and torch.equal(rows.double().cpu(), routing.dispatch(x, positions, 74))
    d = torch.randn(74, cols).to(dtype)
    grad, = torch.autograd.grad(rows, on, d.cuda())
    _close("dx", grad, routing.combine(d, positions))
    y_on = y.cuda().requires_grad_()
    out = nn.combine(y_on, r)
    _close("out", out, routing.combine(y, positions, gates))
    d = torch.randn(37, cols).to(dtype)
    dy, dg = torch.autograd.grad(out, [y_on, gates], d.cuda())
    expected, expected_gates = routing.combine_gradient(d, y, positions, gates)
    _close("dy", dy, expected)
    _close("dgates", dg, expected_gates, torch.full_like(expected_gates, cols ** 0.5))


@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 1), (1, 8, 8), (5, 3, 4), (64, 1, 9), (300, 4, 7), (129, 7, 12), (130, 9, 12), (40, 17, 20), (20, 32, 40)])
def test_choices_of_rows(tokens, top_k, experts):
    from viola_amd import nn
    positions, counts, offsets = _places(tokens, experts, top_k, masked=0.1 if tokens > 1 else 0.0, seed=tokens)
    x, y, gates = torch.randn(tokens, 72), torch.randn(tokens * top_k, 72), torch.rand(tokens, top_k)
    r = _routing(positions, offsets, gates.requires_grad_())
    assert torch.equal(nn.dispatch(x.cuda(), r).double().cpu(), routing.dispatch(x, positions, tokens * top_k))
    y_on = y.cuda().requires_grad_()
    out = nn.combine(y_on, r)
    _close("out", out, routing.combine(y, positions, gates))
    d = torch.randn(tokens, 72)
    dy, dg = torch.autograd.grad(out, [y_on, gates], d.cuda())
    expected, expected_gates = routing.combine_gradient(d, y, positions, gates)
    _close("dy", dy, expected)
    _close("dgates", dg, expected_gates, torch.full_like(expected_gates, 72 ** 0.5))
    _close("plain sum", nn.combine(y.cuda(), nn.Routing(r.positions, r.offsets)), routing.combine(y, positions))


def test_fewer_and_more_rows_than_choices():
    from viola_amd import nn
    positions, counts, offsets = _places(50, 8, 2, masked=0.3)
    used = int(counts.sum())
    x = torch.randn(50, 64)
    for rows in (used, used - 7, 0, 100, 130):
        on = x.cuda().requires_grad_()
        r = _routing(positions, offsets)
        out = nn.dispatch(on, r, rows)
        assert torch.equal(out.double().cpu(), routing.dispatch(x, positions, rows))
        d = torch.randn(rows, 64)
        grad, = torch.autograd.grad(out, on, d.cuda())
        _close("dx", grad, routing.combine(d, positions))
        y, gates = torch.randn(rows, 64), torch.rand(50, 2)
        y_on, r = y.cuda().requires_grad_(), _routing(positions, offsets, gates.requires_grad_())
        back = nn.combine(y_on, r)
        _close("out", back, routing.combine(y, positions, gates))
        d = torch.randn(50, 64)
        dy, dg = torch.autograd.grad(back, [y_on, gates], d.cuda())
        expected, expected_gates = routing.combine_gradient(d, y, positions, gates)
        _close("dy", dy, expected)
        _close("dgates", dg, expected_gates, torch.full_like(expected_gates, 8.0))


def test_rows_that_nobody_has_do_not_matter():
    """NaN in rows that no token has reaches neither the sum nor the gates' gradient, and gets no gradient itself."""
    from viola_amd import nn
    positions, counts, offsets = _places(50, 8, 2, masked=0.3)
    used = int(counts.sum())
    y, gates = torch.randn(100, 96), torch.rand(50, 2)
    dirty = y.clone()
    dirty[used:] = math.nan
    r = _routing(positions, offsets, gates.requires_grad_())
    y_on = dirty.cuda().requires_grad_()
    out = nn.combine(y_on, r)
    _close("out", out, routing.combine(y, positions, gates))
    dy, dg = torch.autograd.grad(out.sum(), [y_on, gates])
    assert dy.isfinite().all() and (dy[used:] == 0).all() and dg.isfinite().all()


def test_strided_rows():
    from viola_amd import nn
    positions, counts, offsets = _places(40, 8, 2)
    gates = torch.rand(40, 2)
    r = _routing(positions, offsets, gates)
    for at, width in ((0, 64), (8, 64), (3, 61), (1, 64)):
        wide, wide_y = torch.randn(40, 160), torch.randn(80, 160)
        x, y = wide.cuda()[:, at:at + width], wide_y.cuda()[:, at:at + width]
        assert torch.equal(nn.dispatch(x, r).double().cpu(), routing.dispatch(wide[:, at:at + width], positions, 80))
        _close("out", nn.combine(y, r), routing.combine(wide_y[:, at:at + width], positions, gates))
    x = torch.randn(64, 40).cuda().t()
    assert torch.equal(nn.dispatch(x, r), nn.dispatch(x.contiguous(), r))
    rows = nn.dispatch(torch.randn(4, 10, 64, device="cuda"), r)               # any leading dimensions with as many tokens
    assert rows.shape == (80, 64)


def test_combine_without_one_of_its_gradients():
    from viola_amd import nn
    positions, counts, offsets = _places(30, 8, 2, masked=0.2)
    y, gates, d = torch.randn(60, 64), torch.rand(30, 2), torch.randn(30, 64)
    expected, expected_gates = routing.combine_gradient(d, y, positions, gates)
    y_on = y.cuda().requires_grad_()
    dy, = torch.autograd.grad(nn.combine(y_on, _routing(positions, offsets, gates)), y_on, d.cuda())
    _close("dy", dy, expected)
    g_on = gates.bfloat16().requires_grad_()
    dg, = torch.autograd.grad(nn.combine(y.cuda(), _routing(positions, offsets, g_on)), g_on, d.cuda())
    assert dg.dtype == BF16
    _close("dgates", dg, expected_gates, torch.full_like(expected_gates, 8.0))


def test_offsets_beyond_32_bits():
    """Rows whose elements lie beyond 2^32."""
    from viola_amd import nn
    cols, rows = 1 << 14, (1 << 18) + 5
    positions = torch.tensor([[rows - 1, 0], [rows - 2, 3], [-1, rows - 3]])
    gates = torch.rand(3, 2)
    y = torch.zeros(rows, cols, device="cuda", dtype=BF16)
    for r in positions[positions >= 0].tolist():
        y[r] = torch.randn(cols, device="cuda").bfloat16()
    few = {r: i for i, r in enumerate(sorted(set(positions[positions >= 0].tolist())))}
    small = torch.stack([y[r] for r in few]).cpu()
    mapped = torch.tensor([[few.get(r, -1) for r in row] for row in positions.tolist()])
    routed = _routing(positions, torch.tensor([0, rows]), gates.requires_grad_())
    y.requires_grad_()
    out = nn.combine(y, routed)
    _close("out", out, routing.combine(small, mapped, gates))
    d = torch.randn(3, cols).bfloat16()
    dy, dg = torch.autograd.grad(out, [y, gates], d.cuda())
    expected, expected_gates = routing.combine_gradient(d, small, mapped, gates)
    _close("dy", torch.stack([dy[r] for r in few]), expected)
    _close("dgates", dg, expected_gates, torch.full_like(expected_gates, cols ** 0.5))


def test_refusals():
    from viola_amd import nn
    logits = torch.randn(10, 8, device="cuda")
    experts = torch.zeros(10, 2, dtype=torch.int32, device="cuda")
    x = torch.randn(10, 64, device="cuda")
    r = nn.route(logits, 2)
    for call, match in ((lambda: nn.route(logits, 0), "choices"), (lambda: nn.route(logits, 9), "choices"), (lambda: nn.route(logits.double(), 2), "float32"),
                        (lambda: nn.route(torch.randn(2, 1100, device="cuda"), 2), "1024 experts"), (lambda: nn.route(torch.randn(2, 64, device="cuda"), 33), "choices"),
                        (lambda: nn.route(logits[0], 2), "tokens, experts"), (lambda: nn.route(logits, 2, mask=torch.ones(10, device="cuda")), "mask has to be bool"),
                        (lambda: nn.route(logits, 2, mask=torch.ones(9, dtype=torch.bool, device="cuda")), "mask has to be bool"),
                        (lambda: nn.route(logits, 2, mask=torch.ones(10, dtype=torch.bool)), "mask has to be bool"),
                        (lambda: nn.balance_loss(logits, experts[:9]), "experts have to be"), (lambda: nn.balance_loss(logits, experts.float()), "int32 or int64"),
                        (lambda: nn.dispatch(x[:9], r), "do not belong"), (lambda: nn.dispatch(x, r._replace(positions=r.positions.long())), "int32"),
                        (lambda: nn.dispatch(x, r._replace(offsets=r.offsets.cpu())), "offsets have to be"), (lambda: nn.combine(x[0], r), "rows, features"),
                        (lambda: nn.combine(x, r._replace(gates=r.gates[:9])), "do not belong")):
        with pytest.raises(RuntimeError, match=match):
            call()
    l = logits.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="once only"):
        torch.autograd.grad(nn.route(l, 2).balance, l, create_graph=True)


def test_gates_near_the_end_of_the_normal_numbers():
    """sigmoid(l) itself, element by element: to 2^-21 where it is a normal number, 0 or as good as that below (an exponential is within 2^-22, its reciprocal
    and the product within 2^-24 each)."""
    from viola_amd import nn
    logits = torch.full((2001, 4), -math.inf)
    logits[:, 1] = torch.linspace(-110.0, -75.0, 2001)
    r = nn.route(logits.cuda(), 1, score="sigmoid", normalize=False)
    expected = torch.sigmoid(logits[:, 1].double())
    assert ((r.gates[:, 0].cpu().double() - expected).abs() <= 2.0 ** -21 * expected + 2.0 ** -126).all()
    assert (r.gates[:, 0].cpu()[expected > 2.0 ** -125] > 0).all() and (r.gates >= 0).all()
    again = nn.route(logits.cuda(), 1, score="sigmoid")                       # its share of itself
    assert (again.gates == 1).all()
