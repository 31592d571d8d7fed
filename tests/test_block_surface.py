"""The operators around a block refuse what would not see them, without a GPU: a recorded graph would hold this call's result as a constant."""

import pytest
import torch

I32 = torch.int32


def _calls():
    """name: (function of one float tensor, that tensor)"""
    from viola_amd import nn
    x, logits = torch.randn(4, 8), torch.randn(4, 6)
    places = nn.Routing(torch.zeros(4, 2, dtype=I32), torch.zeros(7, dtype=I32), torch.zeros(4, 2))
    return {
        "norm_before": (lambda t: nn.norm_before(t), x),
        "norm_after": (lambda t: nn.norm_after(t, t), x),
        "norm_between": (lambda t: nn.norm_between(t, t)[1], x),
        "route": (lambda t: nn.route(t, 2).gates, logits),
        "balance_loss": (lambda t: nn.balance_loss(t, torch.zeros(4, 2, dtype=I32))[0], logits),
        "dispatch": (lambda t: nn.dispatch(t, places), x),
        "combine": (lambda t: nn.combine(t, places), x),
    }


NAMES = ("norm_before", "norm_after", "norm_between", "route", "balance_loss", "dispatch", "combine")


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(name):
    f, x = _calls()[name]
    with torch.no_grad(), pytest.raises(NotImplementedError, match="recorded"):
        torch.jit.trace(f, (x,), check_trace=False)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_graphs_are_refused(name, mode):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = _calls()[name]
    with torch.no_grad(), pytest.raises(NotImplementedError):
        make_fx(f, tracing_mode=mode)(x)


@pytest.mark.parametrize("name", NAMES)
def test_fake_tensors_are_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    f, x = _calls()[name]
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError):
        f(x)


@pytest.mark.parametrize("name", NAMES)
def test_transforms_are_refused(name):
    f, x = _calls()[name]
    with pytest.raises(NotImplementedError):
        torch.func.grad(lambda t: f(t).float().sum())(x)
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda t: f(x) * t)(torch.ones(2))


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as forward_ad
    f, x = _calls()[name]
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        f(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", NAMES)
def test_modes_that_watch_are_no_obstacle(name):
    """A dispatch mode of a program's own (a counter of operations) does not see the operators, and they run under it as without: up to the refusal of tensors
    that are not on the GPU here."""
    from torch.utils.flop_counter import FlopCounterMode
    f, x = _calls()[name]
    with FlopCounterMode(display=False), pytest.raises(RuntimeError, match="GPU only"):
        f(x)


def test_a_negative_number_of_rows_is_refused():
    """-1 is no way to ask for the default: a count that went wrong would lay out rows of none."""
    from viola_amd import nn
    places = nn.Routing(torch.zeros(4, 2, dtype=I32), torch.zeros(7, dtype=I32))
    for rows in (-1, -8):
        with pytest.raises(RuntimeError, match="rows is negative"):
            nn.dispatch(torch.randn(4, 8), places, rows)
