"""Products of 8-bit integers with a scale for each token and channel, in 64 bits, with bounds on what 32 bits may make of them. The reference has no such operators:
these are the formulas that the entry points declare (parity unpinned); tests/test_int8_oracle.py holds them to brute force and to differences.

A bound is the sum of what each rounding of the operator can cost: U = 2^-24 for one in 32 bits, relative to the value. Codes are whole numbers: they are the oracle's own
unless a quotient lies so near a half that the error of what is quantized can carry it across; such codes (`loose`) may be one step off."""

import math

import torch

U = 2.0 ** -24
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def gate(g, activation, errors=False):
    """(act(g), act'(g)), with errors also how far each may be off in 32 bits.

    Silu and gelu are g s with s a sigmoid of a = g or a = 2 y, slope = s + g s (1 - s) a'. Three roundings make a gelu's a, which moves s by 3 U |a| relative; the sigmoid itself is
    within 2 ulp (4 U), and below 2^-126 it is 0, as the hardware's exp2 has no subnormal results. 1 - s is off by s's error and one rounding; the products
    and sums are six more."""
    if activation == "relu":
        act, slope = g.clamp(min=0), (g > 0).to(g.dtype)
        return (act, slope, torch.zeros_like(g), torch.zeros_like(g)) if errors else (act, slope)
    if activation == "silu":
        a, inner, moved = g, torch.ones_like(g), 0.0
    else:
        c = 2 * math.sqrt(2 / math.pi)                                       # (1 + tanh y) / 2 = sigmoid(2 y), which does not cancel for y far below zero
        a, inner = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g * g)
        moved = 3 * U * a.abs()
    s, rest = torch.sigmoid(a), torch.sigmoid(-a)
    act, slope = g * s, s + g * s * rest * inner
    if not errors:
        return act, slope
    off = s * (moved + 4 * U) + 2.0 ** -126
    return act, slope, g.abs() * off + U * act.abs(), off + (g.abs() * off * rest + act.abs() * (off + U) + 4 * U * (act * rest).abs()) * inner + U * s + U * slope.abs()


def hidden(x, activation):
    """What is quantized of rows x, and how far 32 bits may be off it."""
    x = x.double()
    if activation is None:
        return x, torch.zeros_like(x)
    g, u = x.chunk(2, -1)
    act, _, off, _ = gate(g, activation, True)
    return act * u, off * u.abs() + U * (act * u).abs()


def quantize(v, off=None):
    """(codes, scale, loose, relative error of the scale) of v's rows; off: how far v may be off."""
    amax = v.abs().amax(-1, keepdim=True)
    scale = (amax / 127).float().double()
    scale = torch.where(torch.isfinite(amax), scale, math.nan)
    q = torch.where(scale > 0, v / scale, 0.0)
    codes = q.round().clamp(-127, 127)
    if off is None or not bool((off > 0).any()):
        return codes, scale, torch.zeros_like(codes, dtype=torch.bool), torch.zeros_like(scale)
    moved = torch.where(amax > 0, off.amax(-1, keepdim=True) / amax, 0.0) + U   # the largest value's error, and another rounding of the quotient
    near = ((q - q.floor()) - 0.5).abs()
    return codes, scale, near <= torch.where(scale > 0, off / scale, 0.0) + q.abs() * moved * 2, moved


def product(quantized, weight, channels, bias=None):
    """(y, bound before y is rounded to its type): weight [n, k] codes"""
    codes, scale, loose, moved = quantized
    w = weight.double()
    sums = (codes @ w.t()) * scale * channels.double()
    y = sums if bias is None else sums + bias.double()
    bound = (3 * U + 2 * moved) * sums.abs() + U * y.abs() + (loose.double() @ w.abs().t()) * scale * channels.double() * (1 + 2.0 ** -10)
    return y, bound + 2.0 ** -148


def forward(x, weight, channels, bias=None, activation=None):
    return product(quantize(*hidden(x, activation)), weight, channels, bias)


def backward(dy, weight, channels, x=None, activation=None):
    """(dx, bound): the gradient as the operator defines it"""
    v = dy.double() * channels.double()
    dh, bound = product(quantize(v, U * v.abs()), weight.t(), torch.ones(weight.shape[1], dtype=torch.float64, device=weight.device))
    if activation is None:
        return dh, bound
    g, u = x.double().chunk(2, -1)
    act, slope, act_off, slope_off = gate(g, activation, True)
    dg, du = dh * u * slope, dh * act
    return torch.cat([dg, du], -1), torch.cat([bound * (u * slope).abs() + slope_off * (dh * u).abs() + 2 * U * dg.abs(),
                                               bound * act.abs() + act_off * dh.abs() + U * du.abs()], -1) * (1 + 2.0 ** -10) + 2.0 ** -140


def within(actual, expected, bound):
    """Whether each value is within its bound, one rounding to its own type on top; NaN where NaN is due."""
    a, e = actual.detach().double(), expected
    both = torch.isnan(a) & torch.isnan(e)
    limit = bound * (1 + UNIT[actual.dtype]) + UNIT[actual.dtype] * e.abs() + TINY[actual.dtype]
    return bool((both | ((a - e).abs() <= limit)).all())
