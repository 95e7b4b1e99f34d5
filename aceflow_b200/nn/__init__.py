from .layers import LayerNorm, Linear, ResidualNorm, RMSNorm, Rotary, SwiGLU
from .module import Module, Parameter
from .retention import MultiScaleRetention

__all__ = ["Module", "Parameter", "Linear", "RMSNorm", "LayerNorm", "ResidualNorm", "Rotary", "SwiGLU",
           "MultiScaleRetention"]
