from .linear import SVDQW4A4Linear, W8A8Linear

__all__ = ["SVDQW4A4Linear", "W8A8Linear"]
