"""Routing of a mixture of experts, beside the variable-group linear that the experts run on: the router's choice with its gates, places,
counts and balance loss (`route`), that loss for choices made elsewhere (`balance_loss`), and the rows' way to the experts and back
(`dispatch`, `combine`). A forward pass can be captured into a graph, a backward pass raises there. The reference has no such operators.

    routing = nn.route(logits, 2)                                   # logits [tokens, experts]
    counts = routing.counts.tolist()                                # grouped_linear takes them on the host
    rows = nn.dispatch(x, routing, sum(counts))
    y = nn.combine(experts(rows, counts), routing)
    loss = task_loss + 0.01 * routing.balance
"""

from typing import NamedTuple, Optional

from torch import Tensor

from .. import _lib


class Routing(NamedTuple):
    """Where tokens go, as `route` gives it; one made by hand needs positions, offsets and, for `combine`, gates.

    positions  [..., chosen] int32: the row of a choice among all rows, which are in the order of the experts and of tokens within one; rows are
               numbered without a gap and none is named twice. Negative: no expert
    offsets    [experts + 1] int32: where each expert's rows begin; the last is the number of rows
    gates      [..., chosen] float32, 0 where there is no expert
    experts    [..., chosen] int32, -1 where there is none
    counts     [experts] int32: rows of each expert
    balance    the balance loss, float32
    """

    positions: Tensor
    offsets: Tensor
    gates: Optional[Tensor] = None
    experts: Optional[Tensor] = None
    counts: Optional[Tensor] = None
    balance: Optional[Tensor] = None


def _score(score):
    if score not in _lib.SCORE:
        raise AssertionError(f"score must be one of {tuple(_lib.SCORE)}, got {score!r}")
    return _lib.SCORE[score]


def _groups(groups):
    if groups < 1:
        raise AssertionError(f"groups must be 1 or more, got {groups!r}")
    return groups


def route(logits, top_k, *, score="softmax", normalize=True, scale=1.0, mask=None, per_sequence=False, bias=None, groups=1, top_groups=None, group_top=1):
    """The `top_k` experts of each token with the largest logits [..., tokens, experts] (ties to the lowest index), as a `Routing`.

    Probabilities are softmax(logits), or with score="sigmoid" sigmoid(logits) over their sum. gates: with `normalize` the chosen ones' share of
    their own sum, otherwise the probability (softmax) or sigmoid(logit) itself, 0 below 2^-126; times `scale`. An expert with a logit of -inf is never chosen. mask
    (bool, [..., tokens]): False for tokens that go nowhere and are not counted. A token whose logits are all -inf is treated like that.

    balance: experts * sum_e (share of the choices that fall on e) * (mean probability of e) over the counted tokens, of the whole batch or
    with `per_sequence` of each sequence (the last but one dimension), then the mean over sequences; 1 where all experts are used alike. Gradients
    flow to the logits from gates and balance. Up to 1024 experts and 32 choices.

    bias [experts]: the choice is by s + bias instead, s being the softmax's probability or sigmoid(logit); gates and balance remain those of s. A program that balances the load
    moves it after each step, for instance by bias += rate * torch.sign(counts.float().mean() - counts); it has no gradient. An expert whose bias is -inf or NaN is never chosen.
    groups: equal runs of experts (up to 64), of which a token's choice is open to the top_groups (all by default) of largest rank, ties to the lower run; a rank is the sum of the
    group_top (1 or 2) largest s + bias of a run; without a bias the choice among their experts is by the logits. Scores are compared as in 64 bits, ties to the lowest index. A row with a NaN logit (with softmax, +inf too) is
    chosen by its logits alone, as without bias and groups."""
    top_groups = groups if top_groups is None else top_groups
    experts, gates, positions, counts, offsets, balance = _lib.host().route(logits, top_k, _score(score), normalize, scale, mask, per_sequence, bias, _groups(groups), top_groups,
                                                                            group_top)
    return Routing(positions, offsets, gates, experts, counts, balance)


def balance_loss(logits, experts, *, score="softmax", mask=None, per_sequence=False):
    """(the balance loss of `route`, counts [experts] int32) for choices made elsewhere: experts [..., tokens, chosen], int32 or int64. An index
    outside of the experts counts nowhere, and no choice of a masked token does."""
    return _lib.host().balance_loss(logits, experts, _score(score), mask, per_sequence)


def dispatch(x, routing, rows=None):
    """The rows of x [..., features] in the order of the experts: [rows, features], each token's once for each expert it goes to. rows: how many to
    lay out, tokens * chosen by default; the sum of the counts where tokens are masked and the experts should not see the rest. Rows that no token
    has are zero; positions from `rows` on are left out (and in `combine` too).

    Places made by hand are taken as they are, since looking at them would wait for the GPU. They stay within the rows whatever they hold, but where they break what
    `Routing` says, values are undefined: of a row that two choices name or that lies at or beyond offsets[-1] (there zeros and tokens are written by one launch), and
    of rows below offsets[-1] that none names (nothing is written there)."""
    return _lib.host().dispatch(x, routing.positions, routing.offsets, rows)


def combine(y, routing):
    """[..., features]: the sum over a token's experts of gate * row of y [rows, features], in 32 bits and of y's type; zero for a token without an
    expert. Gradients flow to y and to the gates; with routing.gates of None the rows are added as they are."""
    return _lib.host().combine(y, routing.positions, routing.offsets, routing.gates)
