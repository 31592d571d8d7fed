"""FP8 modules: Linear, gated MLP, and the variable-group (expert) linear; the norms around a block and the routing to experts;
layers in 8-bit integers."""

from .linear import Linear
from .mlp import MLP
from ._varlen import grouped_linear, GroupedExperts
from ._norm import norm_before, norm_after, norm_between
from ._routing import Routing, route, balance_loss, dispatch, combine
from ._int8 import quantize_int8, int8_linear, int8_grouped_linear, Int8Linear, Int8Experts

__all__ = ["Linear", "MLP", "grouped_linear", "GroupedExperts", "norm_before", "norm_after", "norm_between", "Routing", "route", "balance_loss", "dispatch",
           "combine", "quantize_int8", "int8_linear", "int8_grouped_linear", "Int8Linear", "Int8Experts"]
