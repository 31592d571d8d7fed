"""A small stack of mixture-of-experts blocks trained on synthetic data: norms around each block, a router, FP8 experts.

    python examples/mixture_of_experts.py [steps]

One block is: the norm of the residual stream, a router over it, the rows of the tokens sent to their experts (two FP8 products with a gated
activation between them, one launch for all experts), their results summed under the gates, and the norm, gate and residual sum of that,
fused with the norm of the next block. The balance losses of all blocks are part of the objective.
"""

import sys
from pathlib import Path

import torch
from torch import nn as torch_nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from viola_amd import nn  # noqa: E402


class Experts(torch_nn.Module):
    """Router and gated feed-forward experts of one block."""

    def __init__(self, width, hidden, experts, top_k, device="cuda"):
        super().__init__()
        self.top_k, self.hidden = top_k, hidden
        self.router = torch_nn.Linear(width, experts, bias=False, device=device)
        self.up = nn.GroupedExperts(experts, width, 2 * hidden, device=device)
        self.down = nn.GroupedExperts(experts, hidden, width, device=device)
        # what the optimizer updates; the experts hold FP8 codes of it
        self.masters = [torch_nn.Parameter(e.dequantize_weight()) for e in (self.up, self.down)]
        for i, master in enumerate(self.masters):
            self.register_parameter("master%d" % i, master)

    def forward(self, h, mask=None):
        """h [batch, tokens, width] in BF16 -> (result of the same shape, balance loss, rows of each expert)"""
        routing = nn.route(self.router(h.float()), self.top_k, mask=mask)
        counts = routing.counts.tolist()                                    # the variable-group products take them on the host
        rows = nn.dispatch(h, routing, sum(counts))
        gate, up = self.up(rows, counts).chunk(2, dim=-1)
        rows = self.down(torch_nn.functional.silu(gate) * up, counts)
        return nn.combine(rows, routing), routing.balance, counts

    def lend_gradients(self):
        """Before the optimizer's step: the gradients of the codes are those of their masters."""
        for layer, master in zip((self.up, self.down), self.masters):
            master.grad, layer.weight.grad = layer.weight.grad, None

    def refresh(self):
        """After it: the codes of the new masters."""
        for layer, master in zip((self.up, self.down), self.masters):
            layer.refresh_weight(master)


class Model(torch_nn.Module):
    def __init__(self, width=256, hidden=512, experts=8, top_k=2, blocks=2, device="cuda"):
        super().__init__()
        ones = lambda: torch_nn.Parameter(torch.ones(width, device=device))  # noqa: E731
        self.blocks = torch_nn.ModuleList(Experts(width, hidden, experts, top_k, device) for _ in range(blocks))
        self.before = torch_nn.ParameterList(ones() for _ in range(blocks))
        self.after = torch_nn.ParameterList(ones() for _ in range(blocks))
        self.gate = torch_nn.ParameterList(torch_nn.Parameter(torch.full((width,), 0.3, device=device)) for _ in range(blocks))

    def forward(self, x, mask=None):
        """x [batch, tokens, width], the residual stream in 32 bits -> (the stream after the last block, sum of the balance losses, counts of each block)"""
        balance, counts = 0.0, []
        h = nn.norm_before(x, self.before[0], dtype=torch.bfloat16)
        for i, block in enumerate(self.blocks):
            y, loss, used = block(h, mask)
            balance = balance + loss
            counts.append(used)
            if i + 1 < len(self.blocks):
                x, h = nn.norm_between(x, y, self.after[i], weight=self.before[i + 1], gate=self.gate[i])
            else:
                x = nn.norm_after(x, y, self.after[i], gate=self.gate[i])
        return x, balance, counts


def train(steps=60, batch=8, tokens=128, width=256, lr=2e-3, seed=0):
    """Losses and the balance loss of every step, and the model."""
    torch.manual_seed(seed)
    model = Model(width)
    teacher = torch.randn(width, width, device="cuda") / width ** 0.5
    optimizer = torch.optim.Adam([p for p in model.parameters() if p.dtype == torch.float32], lr=lr)       # the codes follow their masters
    history = []
    for _ in range(steps):
        x = torch.randn(batch, tokens, width, device="cuda")
        target = x + 0.5 * torch.tanh(x @ teacher)
        out, balance, _ = model(x)
        loss = (out - target).square().mean()
        (loss + 0.01 * balance).backward()
        for block in model.blocks:
            block.lend_gradients()
        optimizer.step()
        optimizer.zero_grad()
        for block in model.blocks:
            block.refresh()
        history.append((loss.item(), balance.item() / len(model.blocks)))
    return history, model


if __name__ == "__main__":
    history, model = train(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
    for step in range(0, len(history), max(1, len(history) // 10)):
        print("step %3d  loss %.4f  balance %.3f" % (step, *history[step]))
    with torch.no_grad():                                                   # one token of each of four sequences
        out, _, counts = model(torch.randn(4, 1, 256, device="cuda"))
    print("a step of single tokens:", tuple(out.shape), "rows of the experts:", counts[0])
