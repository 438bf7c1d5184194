from .kernel import backward, forward
from .module import gated_norm

__all__ = ["gated_norm", "forward", "backward"]
