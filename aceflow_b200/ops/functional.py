"""af.ops functional API (mirrors aceflow/ops/functional.py:14-53).

CUDA tensors run in libaceflow_cuda.so; CPU tensors keep the reference's
numpy formulas.  gelu/softmax are off the retention path and CPU-only.
"""
from __future__ import annotations

from typing import Optional

import numpy as np

from ..core.tensor import Tensor


def _ops():
    from .. import cuda_ops

    return cuda_ops


def matmul(a: Tensor, b: Tensor) -> Tensor:
    return a.matmul(b)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    if x.device.is_cuda:
        return Tensor._wrap(_ops().rms_norm(x.torch, weight.torch, eps), x.device)
    arr = x.numpy()
    variance = np.mean(np.square(arr), axis=-1, keepdims=True)
    return Tensor(arr / np.sqrt(variance + eps) * weight.numpy(), x.device)


def residual_norm(x: Tensor, h: Tensor, pre_weight: Tensor, *, post_weight: Optional[Tensor] = None,
                  scale: Optional[Tensor] = None, gate: Optional[Tensor] = None, alpha: float = 1.0,
                  eps: float = 1e-6):
    """The seam between two blocks (an extension, see nn.ResidualNorm): returns
    (z, y), z = alpha * x + scale * swish(gate) * RMSNorm(h) * post_weight and
    y = RMSNorm(z) * pre_weight; what is None is left out."""
    if x.device.is_cuda:
        t = lambda v: None if v is None else v.torch  # noqa: E731
        z, y = _ops().residual_norm(x.torch, h.torch, gate=t(gate), post_w=t(post_weight), scale=t(scale),
                                    pre_w=pre_weight.torch, alpha=alpha, eps=eps)
        return Tensor._wrap(z, x.device), Tensor._wrap(y, x.device)

    def normed(v, w):
        return v / np.sqrt(np.mean(np.square(v), axis=-1, keepdims=True) + eps) * w.numpy()

    n = h.numpy() if post_weight is None else normed(h.numpy(), post_weight)
    if gate is not None:
        g = gate.numpy()
        n = g / (1.0 + np.exp(-g)) * n
    if scale is not None:
        n = scale.numpy() * n
    z = alpha * x.numpy() + n
    return Tensor(z, x.device), Tensor(normed(z, pre_weight), x.device)


def rotary(x: Tensor, inv_freq: Tensor, positions=0, *, layout: str = "interleaved", scale: float = 1.0) -> Tensor:
    """Rotary positions (an extension, see nn.Rotary) on a CUDA tensor
    [B, T, heads, dim] or [rows, heads, dim]; positions as for
    cuda_ops.rotary."""
    if not x.device.is_cuda:
        raise ValueError("ops.rotary takes CUDA tensors; nn.Rotary also runs on the CPU")
    return Tensor._wrap(_ops().rotary(x.torch, inv_freq.torch, positions, layout=layout, scale=scale), x.device)


def swiglu(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor) -> Tensor:
    if x.device.is_cuda:
        ops = _ops()
        gate = ops.linear(x.torch, w_gate.torch)
        up = ops.linear(x.torch, w_up.torch)
        return Tensor._wrap(ops.linear(ops.silu_mul(gate, up), w_down.torch), x.device)
    arr = x.numpy()
    gate = np.matmul(arr, w_gate.numpy().T)
    up = np.matmul(arr, w_up.numpy().T)
    return Tensor(np.matmul(gate / (1.0 + np.exp(-gate)) * up, w_down.numpy().T), x.device)


def silu(x: Tensor) -> Tensor:
    if x.device.is_cuda:
        return Tensor._wrap(_ops().silu_mul(x.torch), x.device)
    arr = x.numpy()
    return Tensor(arr / (1.0 + np.exp(-arr)), x.device)


def gelu(x: Tensor) -> Tensor:
    if x.device.is_cuda:
        raise NotImplementedError("gelu is not part of the retention hot path (no CUDA kernel)")
    arr = x.numpy()
    cdf = 0.5 * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (arr + 0.044715 * np.power(arr, 3))))
    return Tensor(arr * cdf, x.device)


def softmax(x: Tensor, axis: int = -1) -> Tensor:
    if x.device.is_cuda:
        raise NotImplementedError("softmax is not part of the retention hot path (no CUDA kernel)")
    arr = x.numpy()
    e_x = np.exp(arr - np.max(arr, axis=axis, keepdims=True))
    return Tensor(e_x / np.sum(e_x, axis=axis, keepdims=True), x.device)
