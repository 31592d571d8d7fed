"""Norms around a block with its gate and residual sum, in 64 bits, with the gradients written out. The reference has no such operator:
these are the formulas that the entry points declare (parity unpinned); tests/test_block_operators.py holds the gradients to central differences.

    out = rho x + alpha g (n(y) w_a + b_a)          after=None: n(y) is y
    h   = (n(out) w_b + b_b) (1 + s) + t

x, y: [rows, cols]; every vector broadcasts against them.
"""

import torch


def _wide(t, like=None):
    return None if t is None else t.detach().double().cpu()


def statistics(v, kind, eps):
    """(deviations from the mean over the row's size, 1 / size)"""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros((), dtype=v.dtype)
    r = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (v - mean) * r, r


def _back(q, hat, r, kind):
    d = q - hat * (q * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - q.mean(-1, keepdim=True)
    return r * d


def norm(x, y=None, after_weight=None, after_bias=None, weight=None, bias=None, gate=None, scale=None, shift=None, *, after="rms", before="rms", residual_scale=1.0,
         branch_scale=1.0, eps=1e-6, dout=None, dh=None):
    """{"out", "h"} and, with dout and / or dh, the gradients of what was given under its own name with a "d" before it, summed to its shape, and
    with an "m" before it the same with every term's magnitude (what rounding errors of a sum are measured by). before=None: no h."""
    given = dict(x=x, y=y, after_weight=after_weight, after_bias=after_bias, weight=weight, bias=bias, gate=gate, scale=scale, shift=shift)
    x, y, w_a, b_a, w_b, b_b, g, s, t = (_wide(v) for v in given.values())
    one, zero = torch.ones((), dtype=torch.float64), torch.zeros((), dtype=torch.float64)
    w_a, w_b, g = (one if v is None else v for v in (w_a, w_b, g))
    b_a, b_b, s, t = (zero if v is None else v for v in (b_a, b_b, s, t))
    result = {}
    stream = x
    if y is not None:
        y_hat, y_r = statistics(y, after, eps) if after else (y, one)
        stream = residual_scale * x + branch_scale * g * (y_hat * w_a + b_a)
        result["out"] = stream
    if before:
        x_hat, x_r = statistics(stream, before, eps)
        result["h"] = (x_hat * w_b + b_b) * (1 + s) + t
    if dout is None and dh is None:
        return result
    d = torch.zeros_like(stream) if dout is None else _wide(dout)
    terms = {}
    if dh is not None:
        dh = _wide(dh)
        d = d + _back(dh * (1 + s) * w_b, x_hat, x_r, before)
        terms.update(weight=dh * (1 + s) * x_hat, bias=dh * (1 + s), scale=dh * (x_hat * w_b + b_b), shift=dh)
    terms["x"] = d
    if y is not None:
        terms["x"] = residual_scale * d
        p = branch_scale * d * g * w_a
        terms["y"] = _back(p, y_hat, y_r, after) if after else p
        terms.update(after_weight=branch_scale * d * g * y_hat, after_bias=branch_scale * d * g, gate=branch_scale * d * (y_hat * w_a + b_a))
    for name, v in given.items():
        if v is not None and name in terms:
            term = terms[name].expand(x.shape)
            result["d" + name], result["m" + name] = term.sum_to_size(v.shape), term.abs().sum_to_size(v.shape)
    return result
