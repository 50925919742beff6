"""Graph neural network layers built on the native sparse operators."""
from .attention import AttentionConv
from .conv import SplineConv, GINConv
from .inits import reset, uniform

__all__ = ['AttentionConv', 'SplineConv', 'GINConv', 'reset', 'uniform']
