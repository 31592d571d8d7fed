"""Backward passes of the operators around a block are refused under capture, each by its own node before it launches anything; their forward passes are captured and replayed."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _operators(x, logits, weight):
    """{name: (output, leaf)}; the two of a norm between blocks and the router's two are refused alike"""
    from viola_amd import nn
    r = nn.route(logits, 2)
    rows = nn.dispatch(x, r)
    loss, _ = nn.balance_loss(logits, r.experts)
    return {"norm_before": (nn.norm_before(x, weight), x), "norm_after": (nn.norm_after(x, x, weight), weight), "gates": (r.gates, logits), "balance": (r.balance, logits),
            "balance_loss": (loss, logits), "dispatch": (rows, x), "combine": (nn.combine(rows, r), x)}


def test_captured_backward_passes_are_refused():
    """No eager graph of these leaves is alive, and the capture ends in order."""
    torch.manual_seed(0)
    x, logits = torch.randn(40, 64, device="cuda", requires_grad=True), torch.randn(40, 8, device="cuda", requires_grad=True)
    weight = torch.ones(64, device="cuda", requires_grad=True)
    with torch.no_grad():
        ones = {name: torch.ones_like(y) for name, (y, _) in _operators(x, logits, weight).items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _operators(x, logits, weight)
        for name, (y, leaf) in captured.items():
            with pytest.raises(RuntimeError, match="cannot be captured"):
                torch.autograd.grad(y, leaf, ones[name], retain_graph=True)
        captured = {name: y.detach() for name, (y, _) in captured.items()}
    for seed in range(4):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(40, 64))
            logits.copy_(torch.randn(40, 8))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for name, (y, _) in _operators(x, logits, weight).items():
                assert torch.equal(captured[name], y), name
    # eagerly, with the captured graph still there
    for name, (y, leaf) in _operators(x, logits, weight).items():
        grad, = torch.autograd.grad(y, leaf, ones[name], retain_graph=True)
        assert torch.isfinite(grad).all(), name
