"""``t81.nn`` counterpart: the ternary ``Linear`` layer, and the 4-bit layers beside it."""

from .linear import Linear
from .q4 import Q4Experts, Q4Linear
from .sharded import ShardedLinear

__all__ = ["Linear", "Q4Experts", "Q4Linear", "ShardedLinear"]
