"""Norms around a block, fused with the block's gate and residual sum: what a block reads (`norm_before`), what becomes of its result
(`norm_after`), and both in one pass between two blocks (`norm_between`).

    out = residual_scale * x + branch_scale * gate * (n(y) * after_weight + after_bias)
    h   = (n(out) * weight + bias) * (1 + scale) + shift

n divides a row by its root mean square ("rms"), or subtracts its mean first ("layer"). x is the residual stream, y a block's result, h what
the next block reads. Sums and statistics are in 32 bits whatever the types; h is computed from `out` before that is rounded. A
forward pass can be captured into a graph, a backward pass raises there. The reference has no such operator.
"""

from .. import _lib


def _kind(kind, optional=False):
    allowed = ("rms", "layer", None) if optional else ("rms", "layer")
    if kind not in allowed:
        raise AssertionError(f"the kind of norm must be one of {allowed}, got {kind!r}")
    return _lib.NORM[kind]


def norm_before(x, weight=None, bias=None, *, scale=None, shift=None, kind="rms", eps=1e-6, dtype=None):
    """h = (n(x) * weight + bias) * (1 + scale) + shift over the last dimension of x, in `dtype` (x's own by default).

    weight and bias: [features]. scale and shift: [features], or one such vector for each index of x's first dimensions: [batch, features] or
    [batch, 1, features] for x of [batch, tokens, features], [batch, tokens, features] for one a token. Everything may be float32, bfloat16 or
    float16 and have strided rows; all of it has gradients, each of the shape and type of what was given."""
    return _lib.host().norm("norm_before", x, None, None, None, weight, bias, None, scale, shift, 0, _kind(kind), 1.0, 1.0, eps, dtype, False, True)[0]


def norm_after(x, y, weight=None, bias=None, *, gate=None, residual_scale=1.0, branch_scale=1.0, kind="rms", eps=1e-6):
    """residual_scale * x + branch_scale * gate * (n(y) * weight + bias), of x's type; with kind=None n(y) is y.

    x and y: one shape; y may be of another type than x (a 16-bit block on a 32-bit stream). gate: as scale in `norm_before`."""
    return _lib.host().norm("norm_after", x, y, weight, bias, None, None, gate, None, None, _kind(kind, True), 0, residual_scale, branch_scale, eps, None, True, False)[0]


def norm_between(x, y, after_weight=None, after_bias=None, weight=None, bias=None, *, gate=None, scale=None, shift=None, residual_scale=1.0, branch_scale=1.0,
                 after="rms", before="rms", eps=1e-6):
    """(out, h): `norm_after` of one block and `norm_before` of the next in one pass over x and y. out is of x's type, h of y's."""
    out, h = _lib.host().norm("norm_between", x, y, after_weight, after_bias, weight, bias, gate, scale, shift, _kind(after, True), _kind(before), residual_scale,
                              branch_scale, eps, None, True, True)
    return out, h
