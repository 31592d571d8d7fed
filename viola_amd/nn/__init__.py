"""FP8 modules: Linear, gated MLP, and the variable-group (expert) linear; the norms around a block and the routing to experts."""

from .linear import Linear
from .mlp import MLP
from ._varlen import grouped_linear, GroupedExperts
from ._norm import norm_before, norm_after, norm_between
from ._routing import Routing, route, balance_loss, dispatch, combine

__all__ = ["Linear", "MLP", "grouped_linear", "GroupedExperts", "norm_before", "norm_after", "norm_between", "Routing", "route", "balance_loss", "dispatch",
           "combine"]
