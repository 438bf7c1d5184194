from .kernel import backward, decode, forward
from .module import window_attention

__all__ = ["window_attention", "forward", "backward", "decode"]
