from .kernel import backward, forward
from .module import frequencies, rotary

__all__ = ["rotary", "frequencies", "forward", "backward"]
