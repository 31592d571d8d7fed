"""The mixture-of-experts example: norms, router, rows to the FP8 experts and back, and all their gradients, as one model that learns."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "mixture_of_experts.py"
    spec = importlib.util.spec_from_file_location("mixture_of_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_it_learns(example):
    history, _ = example.train(steps=40)
    losses = [loss for loss, _ in history]
    assert all(torch.tensor(history).flatten().isfinite())
    # the target is the input and half of a bounded function of it: a model that adds nothing is off by its variance, which training has to undercut
    assert sum(losses[-5:]) / 5 < 0.8 * losses[0], losses
    assert all(0.9 < balance < 4 for _, balance in history)


def test_tokens_do_not_see_each_other(example):
    """A token alone comes out as in its batch, and masked tokens leave the others as they are: 16-bit rounding of the stream's two updates apart (2^-8
    each of a block's result, gate 0.3)."""
    torch.manual_seed(1)
    model = example.Model()
    x = torch.randn(2, 33, 256, device="cuda")
    mask = torch.rand(2, 33, device="cuda") < 0.7
    with torch.no_grad():
        whole, _, counts = model(x)
        alone, _, _ = model(x[1:, 7:8])
        some, _, fewer = model(x, mask)
    assert (alone[0, 0] - whole[1, 7]).norm() <= 2.0 ** -6 * whole[1, 7].norm()
    assert (some[mask] - whole[mask]).norm() <= 2.0 ** -6 * whole[mask].norm()
    assert torch.equal(some[~mask], x[~mask]) and sum(counts[0]) == 2 * 66 and sum(fewer[0]) == 2 * int(mask.sum())


def test_block_against_plain_products(example):
    """One block against the same sums over all experts in 32 bits, with the weights that the codes stand for: what is left is the FP8 rounding of the rows on the
    way into two products (2^-4 at most of each value, half of that in the 2-norm, twice) and 16-bit rounding."""
    torch.manual_seed(2)
    block = example.Experts(128, 256, 4, 2)
    h = torch.randn(3, 50, 128, device="cuda").bfloat16()
    with torch.no_grad():
        y, balance, counts = block(h)
        p = torch.softmax(block.router(h.float()), -1)
        gates, chosen = p.topk(2, -1)
        gates = gates / gates.sum(-1, keepdim=True)
        plain = torch.zeros(3, 50, 128, device="cuda")
        up, down = block.up.dequantize_weight(), block.down.dequantize_weight()
        for e in range(4):
            g, u = (h.float() @ up[e].t()).chunk(2, -1)
            result = (torch.nn.functional.silu(g) * u) @ down[e].t()
            plain += result * (gates * (chosen == e)).sum(-1, keepdim=True)
    assert counts == torch.bincount(chosen.flatten(), minlength=4).tolist()
    assert (y.float() - plain).norm() <= 2 * 2.0 ** -5 * plain.norm()
