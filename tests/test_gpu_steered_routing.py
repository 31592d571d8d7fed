"""nn.route with a bias on the choice and groups of experts, against the 64-bit formulas (oracle.routing): choices, places and counts are equal, gates, loss and gradient within
the bounds of tests/test_gpu_routing.py (the same sums)."""

import math

import pytest
import torch

from oracle import routing
from test_gpu_routing import _close, _pull

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _check(logits, top_k, *, bias=None, groups=1, top_groups=None, group_top=1, score="sigmoid", mask=None, normalize=True, scale=1.0, per_sequence=False, on=None):
    from viola_amd import nn
    torch.manual_seed(3)
    top_groups = groups if top_groups is None else top_groups
    l = (logits.cuda() if on is None else on).detach().requires_grad_()
    r = nn.route(l, top_k, score=score, normalize=normalize, scale=scale, mask=None if mask is None else mask.cuda(), per_sequence=per_sequence,
                 bias=None if bias is None else bias.cuda(), groups=groups, top_groups=top_groups, group_top=group_top)
    chosen = routing.choose_steered(logits, top_k, score, mask, bias, groups, top_groups, group_top)
    positions, counts, offsets = routing.places(chosen, logits.shape[-1])
    for name, t, e in (("experts", r.experts, chosen), ("positions", r.positions, positions), ("counts", r.counts, counts), ("offsets", r.offsets, offsets)):
        assert t.dtype == torch.int32 and torch.equal(t.cpu().long(), e), name
    if not bool(torch.isfinite(logits).all()):
        return r
    _close("gates", r.gates, routing.gates(logits, chosen, score, normalize, scale))
    loss, _, _ = routing.balance(logits, chosen, score, mask, per_sequence)
    _close("balance", r.balance, loss)
    dgates, dloss = torch.randn(r.gates.shape), 1.5
    grad, = torch.autograd.grad([r.gates, r.balance], l, [dgates.cuda(), torch.tensor(dloss, device="cuda")])
    assert grad.dtype == l.dtype
    _close("dlogits", grad, routing.gradient(logits, chosen, score, mask, per_sequence, dloss=dloss, dgates=dgates, normalize=normalize, scale=scale),
           _pull(logits, chosen, score, mask, per_sequence, dloss, dgates, normalize, scale))
    return r


def _bias(experts, score, size=0.1):
    return torch.randn(experts) * (size if score == "sigmoid" else size / experts)


@pytest.mark.parametrize("experts", [1, 2, 3, 8, 9, 16, 31, 32, 60, 64, 100, 128, 160, 256, 257, 384, 512, 700, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_bias(experts, score):
    torch.manual_seed(experts)
    _check(torch.randn(70, experts) * 2, min(experts, 4), bias=_bias(experts, score), score=score)


@pytest.mark.parametrize("experts,groups,top_groups", [(4, 2, 1), (8, 4, 2), (8, 8, 3), (12, 4, 2), (15, 5, 2), (16, 8, 3), (32, 16, 5), (60, 6, 3), (64, 8, 3), (64, 64, 9), (96, 3, 2),
                                                       (128, 64, 7), (160, 8, 3), (256, 8, 4), (256, 32, 5), (384, 12, 4), (512, 64, 8), (700, 7, 3), (1024, 16, 4)])
@pytest.mark.parametrize("score,biased,group_top", [("sigmoid", True, 2), ("sigmoid", True, 1), ("sigmoid", False, 2), ("softmax", False, 1), ("softmax", True, 2), ("softmax", False, 2)])
def test_groups(experts, groups, top_groups, score, biased, group_top):
    torch.manual_seed(experts + groups)
    size = experts // groups
    _check(torch.randn(45, experts) * 1.5, min(6, top_groups * size), bias=_bias(experts, score) if biased else None, groups=groups, top_groups=top_groups,
           group_top=min(group_top, size), score=score)


@pytest.mark.parametrize("top_k", [1, 2, 3, 5, 8, 13, 32])
@pytest.mark.parametrize("score,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_choices(top_k, score, normalize):
    torch.manual_seed(top_k)
    _check(torch.randn(90, 64), top_k, bias=_bias(64, score), groups=4, top_groups=2, group_top=2, score=score, normalize=normalize, scale=2.5)


@pytest.mark.parametrize("top_k", [32])
@pytest.mark.parametrize("experts", [512, 1024])
def test_the_most_of_everything(experts, top_k):
    torch.manual_seed(5)
    _check(torch.randn(300, experts), top_k, bias=_bias(experts, "sigmoid"), groups=64, top_groups=16, group_top=2)


@pytest.mark.parametrize("shape", [(1, 64), (2, 64), (31, 8), (257, 8), (300, 3), (32, 64), (33, 64), (1000, 16), (4099, 12), (2, 2, 64), (3, 129, 64), (16, 77, 8), (300, 2, 4), (600, 1, 5),
                                   (3, 4, 5, 64)])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_tokens_and_sequences(shape, per_sequence):
    torch.manual_seed(shape[0])
    even = shape[-1] % 4 == 0
    _check(torch.randn(shape), min(2, shape[-1]), bias=_bias(shape[-1], "sigmoid"), groups=4 if even else 1, top_groups=2 if even else 1, per_sequence=per_sequence)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("experts", [16, 60, 64])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties(dtype, experts, score):
    """Logits on a coarse grid: experts and groups tie in most rows; with a bias that is a multiple of one step, sums tie that are made of different parts."""
    torch.manual_seed(4)
    logits = (torch.randn(200, experts) * 2).round().div(2).to(dtype)
    for bias in (None, torch.zeros(experts), torch.randint(-2, 3, (experts,)) * 0.25):
        for group_top in (1, 2):
            _check(logits, 6, bias=bias, groups=4, top_groups=2, group_top=group_top, score=score)


def test_scores_that_32_bits_cannot_tell_apart():
    """Biases that bring scores to within a few units of the last place of 64 bits' reach: the order is that of 64 bits, in every row."""
    torch.manual_seed(6)
    for score in ("sigmoid", "softmax"):
        logits = torch.randn(1, 32).expand(400, 32).clone() + torch.randn(400, 1) * 1e-3
        s = torch.sigmoid(logits[0].double()) if score == "sigmoid" else torch.softmax(logits[0].double(), -1)
        bias = (s.mean() - s + torch.randn(32) * 1e-9).float()               # all sums nearly alike
        _check(logits, 5, bias=bias, groups=4, top_groups=2, group_top=2, score=score)
        _check(logits, 5, bias=bias, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_far_logits(score):
    torch.manual_seed(8)
    for scale, shift in ((30.0, 0.0), (1.0, 500.0), (1.0, -90.0), (1e-4, 0.0)):
        _check(torch.randn(40, 64) * scale + shift, 4, bias=_bias(64, score), groups=8, top_groups=3, group_top=2, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_tokens_and_closed_experts(score):
    torch.manual_seed(7)
    logits = torch.randn(6, 50, 48)
    logits[0, :, :12] = -math.inf                                            # a whole group
    logits[1, 3] = -math.inf                                                 # a whole row
    logits[2, :, 5:] = -math.inf                                             # fewer experts than choices
    logits[3, 4, 7] = math.nan
    logits[3, 5, 9] = math.inf
    bias = _bias(48, score)
    bias[20], bias[21], bias[30] = -math.inf, math.nan, 5.0
    mask = torch.rand(6, 50) < 0.7
    for options in (dict(bias=bias), dict(bias=bias, groups=4, top_groups=2, group_top=2), dict(groups=4, top_groups=2, group_top=2), dict(groups=4, top_groups=1)):
        r = _check(logits, 7, mask=mask, score=score, **options)
        assert (r.experts[~mask.cuda()] == -1).all() and (r.gates[~mask.cuda()] == 0).all()
    r = _check(logits[4:], 7, mask=mask[4:], score=score, bias=bias, groups=4, top_groups=2, group_top=2, per_sequence=True)
    assert not ((r.experts == 20) | (r.experts == 21)).any()


def test_infinite_bias():
    torch.manual_seed(9)
    bias = _bias(64, "sigmoid")
    bias[[3, 40]] = math.inf
    _check(torch.randn(50, 64), 4, bias=bias)
    _check(torch.randn(50, 64), 4, bias=bias, groups=8, top_groups=2, group_top=2)


def test_types_of_bias_and_strided_logits():
    torch.manual_seed(10)
    wide = torch.randn(60, 100)
    for dtype in (F32, BF16, F16):
        bias = _bias(64, "sigmoid").to(dtype)
        _check(wide[:, 3:67], 4, bias=bias, groups=8, top_groups=3, on=wide.cuda()[:, 3:67])
    _check(wide[:, :64], 4, bias=torch.stack([bias, bias], 1)[:, 0], on=wide.cuda()[:, :64])


def test_all_groups_open_and_no_bias_is_the_plain_choice():
    from viola_amd import nn
    torch.manual_seed(11)
    logits = torch.randn(500, 64, device="cuda")
    plain = nn.route(logits, 4)
    for options in (dict(groups=8), dict(groups=8, top_groups=8, group_top=2), dict(groups=1, top_groups=1)):
        for a, b in zip(nn.route(logits, 4, **options), plain):
            assert torch.equal(a, b)
    steered = nn.route(logits, 4, bias=torch.zeros(64, device="cuda"))
    assert torch.equal(steered.experts, plain.experts) and torch.equal(steered.positions, plain.positions) and torch.equal(steered.gates, plain.gates)


def test_no_tokens_and_no_gradient_for_the_bias():
    from viola_amd import nn
    bias = torch.zeros(8, device="cuda")
    r = nn.route(torch.zeros(0, 8, device="cuda"), 2, bias=bias, groups=2, top_groups=1)
    assert r.experts.shape == (0, 2) and (r.counts == 0).all() and (r.offsets == 0).all()
    logits = torch.randn(5, 8, device="cuda")
    for options in (dict(bias=bias.clone().requires_grad_()), dict(bias=bias[:7]), dict(bias=bias.cpu()), dict(bias=bias.double()), dict(groups=3), dict(groups=128), dict(groups=4, top_groups=0),
                    dict(groups=4, top_groups=5), dict(groups=4, group_top=3), dict(groups=8, top_groups=2, group_top=2), dict(groups=8, top_groups=1)):
        with pytest.raises(RuntimeError):
            nn.route(logits, 2, **options)
    with pytest.raises(AssertionError):
        nn.route(logits, 2, groups=0)


def test_replayed_choice_follows_bias_and_logits():
    from viola_amd import nn
    torch.manual_seed(12)
    logits, bias = torch.randn(700, 128, device="cuda"), torch.zeros(128, device="cuda")

    def step():
        with torch.no_grad():
            return nn.route(logits, 8, score="sigmoid", bias=bias, groups=8, top_groups=4, group_top=2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        logits.copy_(torch.randn(700, 128))
        bias.add_(0.05 * torch.sign(captured.counts.float().mean() - captured.counts))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_large_batches_are_chosen_as_small_ones():
    """Blocks, stages and the rare rows of 64 bits: every row alone gives the same experts."""
    from viola_amd import nn
    torch.manual_seed(13)
    for experts, dtype in ((256, F32), (64, BF16), (16, BF16)):
        logits = (torch.randn(20000, experts, device="cuda") * 1.2).to(dtype)
        bias = torch.randn(experts, device="cuda") * 0.02
        for score in ("sigmoid", "softmax"):
            options = dict(score=score, bias=bias if score == "sigmoid" else bias / experts, groups=8, top_groups=4, group_top=2)
            r = nn.route(logits, 6, **options)
            parts = torch.cat([nn.route(part, 6, **options).experts for part in logits.split(777)])
            assert torch.equal(parts, r.experts)
            l = logits.double()
            c = (torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1)) + options["bias"].double()
            rank = c.view(-1, 8, experts // 8).topk(2, -1).values.sum(-1)
            kept = torch.zeros_like(rank).scatter_(-1, torch.sort(rank, descending=True, stable=True).indices[:, :4], 1.0)
            c = torch.where(kept.repeat_interleave(experts // 8, -1) > 0, c, -math.inf)
            assert torch.equal(torch.sort(c, descending=True, stable=True).indices[:, :6].int(), r.experts)


@pytest.mark.parametrize("far", [-86.0, -100.0, -300.0])
@pytest.mark.parametrize("experts,groups", [(8, 1), (32, 4), (256, 8), (600, 1)])
def test_scores_below_the_smallest_float(far, experts, groups):
    """Sigmoids that 32 bits cannot hold beside biases of zero, or of next to nothing, are ordered in 64."""
    torch.manual_seed(14)
    logits = far + torch.randn(50, experts)
    for bias in (torch.zeros(experts), -torch.zeros(experts), torch.randint(-3, 4, (experts,)) * 2.0 ** -149, torch.randn(experts) * 2.0 ** -130):
        _check(logits, min(6, experts), bias=bias, groups=groups, top_groups=max(1, groups // 2), group_top=2)
