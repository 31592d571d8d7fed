"""Operators around a block without a GPU: the 64-bit formulas that the GPU tests compare with (gradients against central differences, choices and
places by brute force), and what the entry points and the Python operators refuse."""

import itertools
import math
from pathlib import Path

import pytest
import torch

from oracle import norms, routing


# ---------------------------------------------------------------------------------------------------------- the formulas
def _differences(f, t, step=1e-5):
    """Central differences of a scalar function in every element of t."""
    grad = torch.zeros_like(t)
    for i in range(t.numel()):
        up, down = t.clone(), t.clone()
        up.view(-1)[i] += step
        down.view(-1)[i] -= step
        grad.view(-1)[i] = (f(up) - f(down)) / (2 * step)
    return grad


@pytest.mark.parametrize("after,before", itertools.product(("rms", "layer", None), ("rms", "layer", None)))
def test_norm_gradients_are_those_of_differences(after, before):
    torch.manual_seed(1)
    b, s, c = 2, 3, 5
    r = lambda *shape: torch.randn(*shape, dtype=torch.float64)  # noqa: E731
    given = dict(x=r(b, s, c), y=r(b, s, c), after_weight=r(c), after_bias=r(c), gate=r(b, 1, c))
    if before:
        given.update(weight=r(c), bias=r(c), scale=r(b, 1, c), shift=r(b, 1, c))
    options = dict(after=after, before=before, residual_scale=0.7, branch_scale=1.3, eps=1e-3)
    dout, dh = r(b, s, c), r(b, s, c) if before else None

    def loss(**changed):
        out = norms.norm(**{**given, **changed}, **options)
        return (out["out"] * dout).sum() + ((out["h"] * dh).sum() if before else 0.0)

    result = norms.norm(**given, **options, dout=dout, dh=dh)
    for name, t in given.items():
        expected = _differences(lambda v: loss(**{name: v}), t)
        assert (result["d" + name] - expected).abs().max() < 1e-7 * max(1.0, expected.abs().max()), name


@pytest.mark.parametrize("score,normalize,per_sequence", itertools.product(("softmax", "sigmoid"), (True, False), (True, False)))
def test_routing_gradients_are_those_of_differences(score, normalize, per_sequence):
    torch.manual_seed(2)
    logits = torch.randn(2, 4, 6, dtype=torch.float64)
    logits[0, 1, 3] = -math.inf
    mask = torch.tensor([[True, True, True, False], [True, True, False, True]])
    chosen = routing.choose(logits, 3, mask)
    dgates = torch.randn(2, 4, 3, dtype=torch.float64)

    def loss(l):
        return 1.7 * routing.balance(l, chosen, score, mask, per_sequence)[0] + (dgates * routing.gates(l, chosen, score, normalize, 2.0)).sum()

    grad = routing.gradient(logits, chosen, score, mask, per_sequence, dloss=1.7, dgates=dgates, normalize=normalize, scale=2.0)
    finite = torch.isfinite(logits)
    expected = torch.zeros_like(logits)
    for i in finite.view(-1).nonzero()[:, 0].tolist():
        step = torch.zeros(logits.numel(), dtype=torch.float64)
        step[i] = 1e-5
        expected.view(-1)[i] = (loss(logits + step.view(logits.shape)) - loss(logits - step.view(logits.shape))) / 2e-5
    assert (grad - expected)[finite].abs().max() < 1e-8
    assert (grad[~finite] == 0).all() and (grad[~mask] == 0).all()


def test_balance_of_an_even_router_is_one():
    logits = torch.zeros(6, 4)
    chosen = torch.tensor([[0, 1], [2, 3], [0, 2], [1, 3], [0, 3], [1, 2]])
    loss, counts, _ = routing.balance(logits, chosen, "softmax")
    assert abs(loss - 1) < 1e-12 and counts.tolist() == [3, 3, 3, 3]


def test_choice_and_places_by_hand():
    logits = torch.tensor([[1.0, 1.0, 0.0], [-math.inf, 2.0, -math.inf], [math.nan, 3.0, math.inf], [-0.0, 0.0, -1.0]])
    chosen = routing.choose(logits, 2)
    assert chosen.tolist() == [[0, 1], [1, -1], [0, 2], [0, 1]]
    positions, counts, offsets = routing.places(chosen, 3)
    assert counts.tolist() == [3, 3, 1] and offsets.tolist() == [0, 3, 6, 7]
    assert positions.tolist() == [[0, 3], [4, -1], [1, 6], [2, 5]]


def test_combine_is_the_adjoint_of_dispatch():
    torch.manual_seed(3)
    chosen = routing.choose(torch.randn(7, 5), 2, torch.rand(7) < 0.8)
    positions, counts, _ = routing.places(chosen, 5)
    x, d = torch.randn(7, 3, dtype=torch.float64), torch.randn(14, 3, dtype=torch.float64)
    assert torch.isclose((routing.dispatch(x, positions, 14) * d).sum(), (x * routing.combine(d, positions)).sum())
    gates, y = torch.rand(7, 2, dtype=torch.float64), torch.randn(14, 3, dtype=torch.float64)
    dout = torch.randn(7, 3, dtype=torch.float64)
    dy, dg = routing.combine_gradient(dout, y, positions, gates)
    expected = _differences(lambda v: (routing.combine(y, positions, v) * dout).sum(), gates)
    assert (dg - expected).abs().max() < 1e-8
    assert torch.isclose((dy * y).sum(), (routing.combine(y, positions, gates) * dout).sum())


# ---------------------------------------------------------------------------------------------------------- refusals
P = 0x10000                                                                # an aligned address that is never touched
F32, BF16, E4M3 = 0, 1, 3


def _norm_forward(**changed):
    from viola_amd import _lib
    a = dict(x=P, x_pitch=64, x_dtype=BF16, y=P, y_pitch=64, branch=BF16, rows=8, cols=64, after=1, aw=None, ab=None, before=1, w=None, b=None, weight=F32, gate=None,
             gate_pitch=0, scale=None, scale_pitch=0, shift=None, shift_pitch=0, vector=F32, group=8, rho=1.0, alpha=1.0, eps=1e-6, out=P, h=P, stats=None, stream=None)
    return _lib.library().viola_norm_forward(*{**a, **changed}.values())


def test_norm_entry_points_refuse_what_no_kernel_takes():
    assert _norm_forward(rows=0) == 0
    assert _norm_forward(x_dtype=E4M3) == -1 and _norm_forward(branch=E4M3) == -1 and _norm_forward(weight=E4M3) == -1 and _norm_forward(vector=7) == -1
    assert _norm_forward(after=3) == -1 and _norm_forward(before=-1) == -1 and _norm_forward(eps=-1.0) == -1
    assert _norm_forward(x=None) == -1 and _norm_forward(x_pitch=63) == -1 and _norm_forward(y_pitch=63) == -1
    assert _norm_forward(out=None) == -1                                    # y without out
    assert _norm_forward(y=None) == -1                                      # out without y
    assert _norm_forward(h=None) == -1                                      # a norm before the next block without h
    assert _norm_forward(before=0) == -1                                    # h without a norm
    assert _norm_forward(group=3) == -1 and _norm_forward(group=0) == -1    # rows that are no whole groups
    assert _norm_forward(gate=P, gate_pitch=32) == -1                       # overlapping vectors
    assert _norm_forward(stats=P + 8) == -1                                 # statistics not 16-byte aligned
    assert _norm_forward(cols=0) == -1 and _norm_forward(rows=-1) == -1


def test_norm_portions():
    from viola_amd import _lib
    portions = _lib.library().viola_norm_portions
    assert portions(0, 8, 1) == 0 and portions(10, 8, 3) == 0 and portions(-1, 8, 1) == 0 and portions(4, 0, 4) == 0
    for cols in (1, 64, 520, 1152, 4096, 5120, 8192, 8200, 20000):
        for rows, group in ((1, 1), (7, 7), (4096, 4096), (4096, 1), (9850, 197), (1 << 20, 1 << 10)):
            count = portions(rows, cols, group)
            assert count % (rows // group) == 0 and rows // group <= count <= rows


def _route(**changed):
    from viola_amd import _lib
    a = dict(logits=P, pitch=16, dtype=F32, tokens=8, experts=16, top_k=2, score=0, normalize=1, scale=1.0, mask=None, sequence=8, chosen=P, gates=P, positions=P, counts=P,
             offsets=P, loss=P, cost=P, stats=None, workspace=P, words=1 << 20, stream=None)
    return _lib.library().viola_route_forward(*{**a, **changed}.values())


def test_route_entry_points_refuse_what_no_kernel_takes():
    from viola_amd import _lib
    assert _route(tokens=0) == 0
    assert _route(dtype=E4M3) == -1 and _route(score=2) == -1 and _route(pitch=15) == -1 and _route(top_k=0) == -1 and _route(top_k=17) == -1
    assert _route(sequence=3) == -1 and _route(sequence=0) == -1 and _route(words=10) == -1 and _route(workspace=None) == -1 and _route(gates=None) == -1
    assert _route(experts=1025, pitch=1025) == -2 and _route(experts=64, pitch=64, top_k=33) == -2 and _route(tokens=1 << 30, sequence=1 << 30) == -1
    assert _route(stats=P + 4) == -1
    words = _lib.library().viola_route_workspace
    assert words(0, 16, 8) == 0 and words(8, 0, 8) == 0 and words(8, 16, 3) == 0 and words(8, 1025, 8) == 0
    assert words(8, 16, 8) == 2 * 16 + 1                                    # one portion: its sums, counts and tokens


def test_rows_entry_points_refuse_what_no_kernel_takes():
    from viola_amd import _lib
    lib = _lib.library()
    gather = lambda rows=P, pitch=64, count=16, dtype=BF16, cols=64, positions=P, tokens=8, top_k=2, out=P: lib.viola_rows_gather(  # noqa: E731
        rows, pitch, count, dtype, cols, positions, None, tokens, top_k, out, None)
    assert gather(tokens=0) == 0
    assert gather(dtype=E4M3) == -1 and gather(pitch=63) == -1 and gather(cols=0) == -1 and gather(out=None) == -1 and gather(positions=None) == -1
    assert gather(top_k=0) == -1 and gather(rows=None) == -1 and gather(tokens=1 << 31) == -1 and gather(count=1 << 31) == -1
    scatter = lambda x=P, pitch=64, dtype=BF16, cols=64, positions=P, tokens=8, top_k=2, rows=P, count=16, values=None, values_pitch=0, dots=None: (  # noqa: E731
        lib.viola_rows_scatter(x, pitch, dtype, cols, positions, None, tokens, top_k, P, rows, count, values, values_pitch, dots, None))
    assert scatter(tokens=0) == 0
    assert scatter(dtype=E4M3) == -1 and scatter(pitch=63) == -1 and scatter(x=None) == -1 and scatter(rows=None) == -1
    assert scatter(dots=P) == -1 and scatter(dots=P, values=P, values_pitch=63) == -1


def test_operators_refuse_on_the_host():
    from viola_amd import nn
    x, logits = torch.randn(4, 8), torch.randn(4, 6)
    with pytest.raises(RuntimeError, match="GPU only"):
        nn.norm_before(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        nn.norm_between(x, x)
    with pytest.raises(AssertionError, match="kind of norm"):
        nn.norm_before(x, kind="batch")
    with pytest.raises(AssertionError, match="kind of norm"):
        nn.norm_before(x, kind=None)
    with pytest.raises(AssertionError, match="score must be"):
        nn.route(logits, 2, score="linear")
    with pytest.raises(RuntimeError, match="GPU only"):
        nn.route(logits, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        nn.balance_loss(logits, torch.zeros(4, 2, dtype=torch.int32))
    places = nn.Routing(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(7, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        nn.dispatch(x, places)
    with pytest.raises(RuntimeError, match="GPU only"):
        nn.combine(x, places)


def test_sizes_beyond_the_limits_have_no_workspace():
    """Asked beyond what the entry points take, the two sizes are 0: no division by what an overflow left, which ends the process."""
    import subprocess
    import sys
    program = """if True:
        from viola_amd import _lib
        words, portions = _lib.library().viola_route_workspace, _lib.library().viola_norm_portions
        assert words((1 << 26) - 1, 16, (1 << 26) - 1) > 0 and portions(8, 1 << 28, 8) == 8
        for experts in (4, 16, 128, 1024):
            for bits in range(26, 63):
                assert words(1 << bits, experts, 1 << bits) == 0 and words(1 << bits, experts, 1) == 0, (experts, bits)
        for bits in range(29, 63):
            assert portions(8, 1 << bits, 8) == 0 and portions(8, (1 << bits) + 1, 1) == 0, bits"""
    done = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
