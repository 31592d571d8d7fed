"""Layers in 8-bit integers, with a scale for each token and each channel: weights are fixed codes, tokens are quantized on the way in.

    y = (q @ weight.T) * s * weight_scale + bias        q, s = quantize_int8(x): s = max|row| / 127, q = round(row / s)

The sum over the features is exact, the scales are applied in 32 bits, and the result is rounded once. With an activation x is [g | u], what a projection to both branches
of a gated block gives, and act(g) * u is quantized (gelu is its tanh form, as in `MLP`).

Gradients flow to x and bias as if rounding to integers were the identity, and the gradient is a product of the same kind: dx = (q' @ weight) * s' with
q', s' = quantize_int8(dy * weight_scale). So adapters, norms and routers beside fixed layers can be trained through them. A forward pass can be
captured into a graph, a backward pass raises there. The reference has no such operators.

    up, down = nn.Int8Experts.from_float(fp8_up), nn.Int8Experts.from_float(fp8_down, activation="silu")
    routing = nn.route(logits, 8, score="sigmoid", bias=bias, groups=8, top_groups=4, group_top=2)
    y = nn.combine(down(up(nn.dispatch(x, routing), routing.offsets), routing.offsets), routing)         # nothing waits for the GPU
"""

import torch
from torch import nn

from .. import _lib


def _activation(activation):
    if activation is not None and activation not in _lib.ACTIVATION:
        raise AssertionError(f"activation must be None or one of {tuple(_lib.ACTIVATION)}, got {activation!r}")
    return -1 if activation is None else _lib.ACTIVATION[activation]


def quantize_int8(x, *, activation=None):
    """(codes int8, scale float32 [...]) of the rows of x [..., features], or with an activation of act(g) * u for rows [g | u].

    A row of zeros has a scale of 0; one that holds an Inf or a NaN has a scale of NaN and zero codes, so that a product makes all of it NaN. Codes are a view of rows a
    multiple of 16 bytes apart. Of weights [out, in] or [groups, out, in] these are the codes and scales that the products below take. No gradients."""
    return _lib.host().quantize_int8(x, _activation(activation))


def int8_linear(x, weight, weight_scale, bias=None, *, activation=None, dtype=None, weight_t=None):
    """x [..., in] (with an activation [..., 2 in]) through weight int8 [out, in] with weight_scale float32 [out]; of `dtype`, x's own by default.

    weight_t: the transposed codes [in, out] for the gradient of x, made there if it is not given. in (and out, for a gradient) up to 131072; codes whose rows lie a
    multiple of 16 bytes apart are read in place, others are laid out anew by each call."""
    return _lib.host().int8_product("int8_linear", x, weight, weight_scale, bias, None, _activation(activation), dtype, weight_t)


def int8_grouped_linear(x, weight, weight_scale, offsets, *, activation=None, dtype=None, weight_t=None):
    """`int8_linear` for the rows of each group: rows offsets[g] to offsets[g + 1] of x [rows, in] through weight[g] of [groups, out, in] with weight_scale[g] of
    [groups, out]. offsets: int32 [groups + 1] on the GPU, ascending from 0, as `route` gives them, so nothing waits for the counts. Rows from offsets[-1] on are zero, and so are
    their gradients. Offsets made by hand are taken as they are; whatever they hold, a product stays within its rows, but rows that no group or two groups name are undefined."""
    return _lib.host().int8_product("int8_grouped_linear", x, weight, weight_scale, None, offsets, _activation(activation), dtype, weight_t)


class _Fixed(nn.Module):
    """Codes and scales of fixed weights, which `.to()` may move but never cast."""

    def __init__(self, shape, activation, cache_transpose, device):
        super().__init__()
        _activation(activation)
        self.out_features, self.in_features = shape[-2:]
        self.activation, self.cache_transpose = activation, cache_transpose
        pitch = -(-self.in_features // 16) * 16
        self.register_buffer("codes", torch.zeros((*shape[:-1], pitch), dtype=torch.int8, device=device))
        self.register_buffer("weight_scale", torch.zeros(shape[:-1], dtype=torch.float32, device=device))
        self.register_buffer("codes_t", None, persistent=False)

    @property
    def weight(self):
        """int8 [..., out, in]"""
        return self.codes[..., :self.in_features]

    @property
    def weight_t(self):
        """int8 [..., in, out], or None unless it is kept"""
        return None if self.codes_t is None else self.codes_t[..., :self.out_features]

    @torch.no_grad()
    def refresh_weight(self, master):
        """Takes the codes and scales of new weights."""
        if master.shape != self.weight.shape:
            raise AssertionError(f"weights have to be of shape {tuple(self.weight.shape)}, got {tuple(master.shape)}")
        codes, scale = quantize_int8(master)
        self.weight.copy_(codes)
        self.weight_scale.copy_(scale)
        self._turn()

    @torch.no_grad()
    def _turn(self):
        self.codes_t = None
        if self.cache_transpose and self.codes.is_cuda:
            turned = self.weight.transpose(-1, -2)
            self.codes_t = torch.zeros((*turned.shape[:-1], -(-self.out_features // 16) * 16), dtype=torch.int8, device=turned.device)
            self.weight_t.copy_(turned)

    def dequantize_weight(self):
        return self.weight.float() * self.weight_scale[..., None]

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != scale.dtype:                           # cast: moved alone instead (`to_empty` off the meta device has nothing to move)
            self.weight_scale = scale.to(self.weight_scale.device)
        if self.codes_t is None:                                             # loaded on the CPU
            self._turn()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._turn()

    def extra_repr(self):
        shown = dict(in_features=self.in_features, out_features=self.out_features, activation=self.activation, cache_transpose=self.cache_transpose)
        return ", ".join(f"{name}={value!r}" for name, value in shown.items())


class Int8Linear(_Fixed):
    """`int8_linear` with weights of its own: made of another layer by `from_float`, or of zeros until `refresh_weight` or `load_state_dict`. cache_transpose keeps the
    transposed codes for the gradient of x."""

    def __init__(self, in_features, out_features, bias=True, *, activation=None, cache_transpose=False, device=None, dtype=None):
        super().__init__((out_features, in_features), activation, cache_transpose, device)
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None

    @classmethod
    @torch.no_grad()
    def from_float(cls, linear, **options):
        """Of a torch.nn.Linear or an FP8 `Linear` on the GPU."""
        weight = linear.dequantize_weight() if hasattr(linear, "dequantize_weight") else linear.weight
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, device=weight.device, dtype=None if linear.bias is None else linear.bias.dtype, **options)
        layer.refresh_weight(weight)
        if linear.bias is not None:
            layer.bias.copy_(linear.bias)
            layer.bias.requires_grad_(linear.bias.requires_grad)
        return layer

    def forward(self, x):
        return int8_linear(x, self.weight, self.weight_scale, self.bias, activation=self.activation, weight_t=self.weight_t)


class Int8Experts(_Fixed):
    """`int8_grouped_linear` with weights of its own, as `Int8Linear`."""

    def __init__(self, groups, in_features, out_features, *, activation=None, cache_transpose=False, device=None):
        super().__init__((groups, out_features, in_features), activation, cache_transpose, device)
        self.groups = groups

    @classmethod
    @torch.no_grad()
    def from_float(cls, experts, **options):
        """Of `GroupedExperts` on the GPU, or of weights [groups, out, in]."""
        weight = experts.dequantize_weight() if hasattr(experts, "dequantize_weight") else experts
        groups, out_features, in_features = weight.shape
        layer = cls(groups, in_features, out_features, device=weight.device, **options)
        layer.refresh_weight(weight)
        return layer

    def forward(self, x, offsets):
        return int8_grouped_linear(x, self.weight, self.weight_scale, offsets, activation=self.activation, weight_t=self.weight_t)
