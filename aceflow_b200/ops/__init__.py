from .functional import gelu, matmul, residual_norm, rms_norm, rotary, silu, softmax, swiglu

__all__ = ["matmul", "rms_norm", "residual_norm", "rotary", "swiglu", "gelu", "silu", "softmax"]
