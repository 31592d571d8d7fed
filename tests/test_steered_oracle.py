"""oracle.routing's steered choice by hand and beside the plain one, and what its entry point refuses before any launch."""

import math

import pytest
import torch

from oracle import routing


def test_by_hand():
    logits = torch.tensor([[2.0, 1.0, 0.0, 0.5, -1.0, 3.0]])
    bias = torch.tensor([0.0, 0.0, 0.9, 0.0, 0.0, -1.0])
    # sigmoid: .881 .731 .5 .622 .269 .953; with the bias .881 .731 1.4 .622 .269 -.047
    assert routing.choose_steered(logits, 3, "sigmoid", bias=bias).tolist() == [[2, 0, 1]]
    # groups of two: largest .881, 1.4, .269; two largest 1.612, 2.022, .222
    assert routing.choose_steered(logits, 2, "sigmoid", bias=bias, groups=3, top_groups=1).tolist() == [[2, 3]]
    assert routing.choose_steered(logits, 3, "sigmoid", bias=bias, groups=3, top_groups=2, group_top=2).tolist() == [[2, 0, 1]]
    # without a bias the last group has the largest single expert
    assert routing.choose_steered(logits, 2, "sigmoid", groups=3, top_groups=1).tolist() == [[5, 4]]
    assert routing.choose_steered(logits, 2, "sigmoid", groups=3, top_groups=1, group_top=2).tolist() == [[0, 1]]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_without_bias_and_groups_it_is_the_plain_choice(score):
    torch.manual_seed(0)
    logits = (torch.randn(50, 20) * 3).round() / 2
    logits[3, 4], logits[5, 6], logits[7] = math.nan, -math.inf, -math.inf
    logits[9, 2] = math.inf
    mask = torch.rand(50) < 0.8
    assert torch.equal(routing.choose_steered(logits, 4, score, mask), routing.choose(logits, 4, mask))


def test_one_choice_at_a_time():
    """Taking the best, closing it with a bias of -inf, and taking the best again gives the same order."""
    torch.manual_seed(1)
    logits, bias = torch.randn(1, 24), torch.randn(24) * 0.1
    whole = routing.choose_steered(logits, 5, "sigmoid", bias=bias)[0].tolist()
    closed, found = bias.clone(), []
    for _ in range(5):
        e = routing.choose_steered(logits, 1, "sigmoid", bias=closed)[0, 0].item()
        found.append(e)
        closed[e] = -math.inf
    assert found == whole


def test_rejected_calls_launch_nothing():
    from viola_amd import _lib
    lib, P = _lib.library(), 0x10000

    def call(**changed):
        a = dict(logits=P, pitch=64, dtype=0, tokens=8, experts=64, top_k=4, score=1, normalize=1, scale=1.0, bias=P, groups=8, top_groups=4, group_top=2, mask=None, sequence=8, chosen=P,
                 gates=P, positions=P, counts=P, offsets=P, loss=P, cost=P, stats=P, workspace=P, words=1 << 20, stream=None)
        return lib.viola_route_steered_forward(*{**a, **changed}.values())

    for bad in (dict(groups=0), dict(groups=7), dict(top_groups=0), dict(top_groups=9), dict(group_top=0), dict(group_top=3), dict(groups=64, group_top=2), dict(groups=64, top_groups=3, group_top=1),
                dict(dtype=3), dict(score=2), dict(tokens=-8), dict(sequence=3), dict(pitch=63), dict(words=0), dict(workspace=P + 4), dict(chosen=None), dict(cost=None)):
        assert call(**bad) == -1, bad
    assert call(experts=1024, pitch=1024, groups=128) == -2 and call(experts=2048, pitch=2048) == -2 and call(top_k=33) == -2
    assert call(tokens=0, sequence=1) == 0
    for tokens, experts, sequence in ((1, 8, 1), (5000, 256, 5000), (32768, 256, 2048), (4096, 1024, 1), (100000, 16, 100000)):
        assert lib.viola_route_steered_workspace(tokens, experts, sequence) > 0
    assert lib.viola_route_steered_workspace(0, 8, 1) == 0 and lib.viola_route_steered_workspace(8, 2000, 8) == 0
