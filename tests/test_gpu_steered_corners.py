"""Corners of nn.route with a bias and groups, against the 64-bit formulas: choices equal, gates, loss and gradient within the bounds of tests/test_gpu_steered_routing.py."""

import math

import pytest
import torch

from oracle import routing
from test_gpu_steered_routing import _bias, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [8, 60, 64, 256, 700])
@pytest.mark.parametrize("top_k", [1, 3, 6])
def test_chosen_experts_far_below_the_largest(score, experts, top_k):
    """A bias of -inf closes each row's likely experts; the gates are the shares of what is left, however small its scores are beside those."""
    torch.manual_seed(experts)
    bias = _bias(experts, score, 1e-3)
    bias[:2] = -math.inf
    for far in (-60.0, -100.0, -300.0):
        logits = far + 8 * torch.randn(70, experts)
        logits[:50, 0] = torch.randn(50)
        logits[20:60, 1] = 1.0
        _check(logits, top_k, bias=bias, score=score)                        # (the last rows have no likely expert)
        _check(logits, min(top_k, experts // 2), bias=bias, score=score, groups=4, top_groups=2, group_top=2, scale=2.5)
        coarse = (logits / 4).round() * 4                                    # ties: rows that are chosen again in 64 bits
        _check(coarse, top_k, bias=torch.where(bias == -math.inf, bias, 0.0), score=score)
        _check(coarse, top_k, bias=bias, score=score, mask=torch.rand(70) < 0.7)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_no_expert_left(score):
    from viola_amd import nn
    torch.manual_seed(1)
    logits = torch.randn(40, 16)
    logits[:, 3:] -= 200.0
    bias = torch.full((16,), -math.inf)
    r = _check(logits, 2, bias=bias, score=score)
    assert (r.experts == -1).all() and (r.gates == 0).all()
    bias[7] = 0.0
    l = logits.cuda().requires_grad_()
    r = nn.route(l, 2, bias=bias.cuda(), score=score)
    chosen = routing.choose_steered(logits, 2, score, bias=bias)
    assert torch.equal(r.experts.cpu().long(), chosen)
    assert (r.experts[:, 0] == 7).all() and (r.gates[:, 0] == 1).all() and (r.gates[:, 1] == 0).all()
    # a probability below 2^-126 is 0, which costs the loss at most that times the expert's cost, at most the 16 experts over the tokens' number, for each token of each expert
    loss, _, _ = routing.balance(logits, chosen, score)
    assert abs(r.balance.item() - loss.item()) <= 2.0 ** -16 * loss.item() + 16 * 16 * 2.0 ** -126
    grad, = torch.autograd.grad(r.gates, l, torch.ones_like(r.gates))
    assert (grad == 0).all()


def test_groups_apart_by_less_than_the_smallest_normal_number():
    """Sigmoids that 32 bits hold as 0 and biases of a few 2^-149: the order of the groups is that of 64 bits, also where the choices themselves lie far apart."""
    tiny = 2.0 ** -149
    _check(torch.tensor([[-99.0, -100.0, -100.0, -100.0]]), 1, bias=torch.tensor([tiny, -1.0, 2 * tiny, -1.0]), groups=2, top_groups=1)
    _check(torch.tensor([[-100.0, -100.0, -99.0, -100.0]]), 2, bias=torch.tensor([1.0, 3 * tiny, tiny, -1.0]), groups=4, top_groups=2)
    torch.manual_seed(2)
    for experts, groups, group_top in ((8, 2, 1), (32, 8, 1), (64, 16, 2), (256, 8, 2), (1024, 64, 2)):
        size = experts // groups
        for far in (-87.5, -95.0, -102.0):
            bias = -torch.rand(groups, size)
            bias[:, 0] = torch.randint(0, 4, (groups,)) * tiny
            if group_top == 2:                                               # the second of a run the same everywhere
                bias[:, 1] = -2.0 ** -60
                bias[:, 2:] -= 0.5
            _check(far + torch.randn(60, experts), 1, bias=bias.reshape(-1), groups=groups, top_groups=1, group_top=group_top)


def test_ranks_that_only_64_bits_hold():
    """Sums of two biases beyond the largest float: they differ, and are neither infinite nor those of closed runs."""
    torch.manual_seed(3)
    low = torch.finfo(torch.float32).min
    for top_groups in (1, 2, 3):
        bias = torch.randn(16)
        bias[:4], bias[4:8], bias[8:12], bias[12:] = -math.inf, low, torch.tensor([low, low, low / 2, low]), low * 0.75
        _check(torch.randn(40, 16), 3, bias=bias, groups=4, top_groups=top_groups, group_top=2)
        bias = torch.zeros(16)
        bias[2:4], bias[4:6], bias[8:10], bias[12:] = 2e38, 3e38, 2.5e38, math.inf
        _check(torch.randn(40, 16), 3, bias=bias, groups=4, top_groups=top_groups, group_top=2)
    bias = torch.zeros(12)
    bias[2:4], bias[4:6], bias[8:10] = 2e38, 3e38, 2.5e38
    for top_groups in (1, 2):
        _check(torch.randn(40, 12), 3, bias=bias, groups=3, top_groups=top_groups, group_top=2)


@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_of_scores_that_are_one_number_in_64_bits(score, group_top):
    """Without a bias, too, runs are ranked by scores as 64 bits hold them, ties to the lower run: sigmoids of large logits, scores of logits next to zero, scores that vanish."""
    if group_top == 1 and score == "sigmoid":
        _check(torch.tensor([[40.0, 1.0, 45.0, 2.0]]), 1, groups=2, top_groups=1)
    for experts, groups in ((8, 4), (16, 4), (64, 8), (60, 6), (256, 8), (256, 64), (1024, 16)):
        torch.manual_seed(experts)
        size = experts // groups
        for scale, shift in ((1.0, 500.0), (30.0, 0.0), (4.0, 24.0), (4.0, 34.0), (1.0, -90.0), (1e-20, 0.0), (1e-20, -1e-18), (300.0, 0.0), (1.0, -1000.0)):
            logits = torch.randn(40, experts) * scale + shift
            logits[:5, 0], logits[3:8, 1::size] = 5.0, -math.inf             # one expert far above the rest in a few rows, experts that are not there in others
            if score == "sigmoid":
                logits[:, 5], logits[7, 3] = 36.0, math.inf
            _check(logits, min(3, size), groups=groups, top_groups=max(1, groups // 3), group_top=min(group_top, size), score=score)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_groups_without_a_bias_at_other_logits(dtype):
    torch.manual_seed(4)
    for score in ("softmax", "sigmoid"):
        for scale in (0.5, 3.0, 8.0):
            _check((torch.randn(200, 512) * scale).to(dtype), 8, groups=64, top_groups=8, group_top=1, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups", [(512, 64, 8), (256, 32, 5), (64, 16, 8), (1024, 64, 31)])
@pytest.mark.parametrize("group_top", [1, 2])
def test_many_groups_of_many_tokens(score, experts, groups, top_groups, group_top):
    """Runs that 32 bits do not order where it matters, among many where it does not; closed runs, and runs that a lowest bias keeps for the last, in every row."""
    from viola_amd import nn
    torch.manual_seed(experts + group_top)
    size = experts // groups
    for deviation in (0.5, 3.0):
        logits = torch.randn(8000, experts, device="cuda") * deviation
        l = logits.double()
        s = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1)
        bias = torch.randn(experts, device="cuda") * (0.02 if score == "sigmoid" else 0.02 / experts)
        closed = bias.clone()
        closed[:size], closed[3 * size:4 * size], closed[5 * size:6 * size] = -math.inf, torch.finfo(torch.float32).min, -math.inf
        for b in (None, bias, closed):
            c = s if b is None else s + b.double()
            rank = c.view(-1, groups, size).topk(group_top, -1).values.sum(-1)
            kept = torch.zeros_like(rank).scatter_(-1, torch.sort(rank, descending=True, stable=True).indices[:, :top_groups], 1.0)
            by = torch.where(kept.repeat_interleave(size, -1) > 0, l if b is None else c, -math.inf)
            r = nn.route(logits, 8, score=score, bias=b, groups=groups, top_groups=top_groups, group_top=group_top)
            assert torch.equal(torch.sort(by, descending=True, stable=True).indices[:, :8].int(), r.experts)
