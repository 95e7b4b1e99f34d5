"""Linear / RMSNorm / LayerNorm / SwiGLU (mirrors aceflow/nn/layers.py:11-88),
and ResidualNorm and Rotary, which the reference lacks.

Initialisation draws from ``np.random`` in the reference's order, so a
seeded script builds identical weights with either package.  On a CUDA
device every forward runs in libaceflow_cuda.so; on the CPU the reference's
numpy formulas apply unchanged.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np

from ..core.tensor import Tensor
from .module import Module, Parameter


def _cuda_ops():
    from .. import cuda_ops

    return cuda_ops


class Linear(Module):
    """Fully connected layer: y = x A^T + b (layers.py:11-33)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        k = 1.0 / math.sqrt(in_features)
        self.weight = Parameter(Tensor(np.random.uniform(-k, k, (out_features, in_features)).astype(np.float32)))
        if bias:
            self.bias = Parameter(Tensor(np.random.uniform(-k, k, (out_features,)).astype(np.float32)))
        else:
            self.bias = None

    def forward(self, x: Tensor) -> Tensor:
        if x.device.is_cuda:
            b = None if self.bias is None else self.bias.torch
            return Tensor._wrap(_cuda_ops().linear(x.torch, self.weight.torch, b), x.device)
        out = np.matmul(x.numpy(), self.weight.numpy().T)
        if self.bias is not None:
            out = out + self.bias.numpy()
        return Tensor(out, x.device)


class RMSNorm(Module):
    """Root Mean Square Layer Normalization (layers.py:36-49), eps 1e-6."""

    def __init__(self, d_model: int, eps: float = 1e-6):
        super().__init__()
        self.d_model = d_model
        self.eps = eps
        self.weight = Parameter(Tensor(np.ones(d_model, dtype=np.float32)))

    def forward(self, x: Tensor) -> Tensor:
        if x.device.is_cuda:
            return Tensor._wrap(_cuda_ops().rms_norm(x.torch, self.weight.torch, self.eps), x.device)
        arr = x.numpy()
        rms = np.sqrt(np.mean(np.square(arr), axis=-1, keepdims=True) + self.eps)
        return Tensor((arr / rms) * self.weight.numpy(), x.device)


class ResidualNorm(Module):
    """The seam between two blocks of a layer: the norm behind a block, its
    gate and residual scale, the residual add and the norm in front of the next
    block (an extension; the reference has the last two alone,
    aceflow-core/src/cpu/mod.rs:672-700):

        n = RMSNorm(h) * post_weight            (with post_norm, else h)
        z = alpha * x + scale * swish(gate) * n  (scale with layer_scale; gate when given)
        y = RMSNorm(z) * pre_weight

    forward(x, h, gate=None) returns (z, y): the residual stream for the next
    seam and the next block's input.  On CUDA it is one kernel
    (af_residual_norm), x and h fp32 or bf16 each (y in h's dtype);
    cuda_ops.residual_norm_autograd is its differentiable form."""

    def __init__(self, d_model: int, eps: float = 1e-6, *, post_norm: bool = True,
                 layer_scale: Optional[float] = None, alpha: float = 1.0):
        super().__init__()
        self.d_model = d_model
        self.eps = eps
        self.alpha = float(alpha)
        self.pre_weight = Parameter(Tensor(np.ones(d_model, dtype=np.float32)))
        self.post_weight = Parameter(Tensor(np.ones(d_model, dtype=np.float32))) if post_norm else None
        self.scale = (None if layer_scale is None
                      else Parameter(Tensor(np.full(d_model, layer_scale, dtype=np.float32))))

    def forward(self, x: Tensor, h: Tensor, gate: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        from ..ops.functional import residual_norm

        return residual_norm(x, h, self.pre_weight, post_weight=self.post_weight, scale=self.scale, gate=gate,
                             alpha=self.alpha, eps=self.eps)


class Rotary(Module):
    """Rotary positions for queries and keys (an extension; RetNet's rotation,
    Sun et al. 2023, eq. 5): turns the first rotary_dim values (all of them by
    default) of every head by position * inv_freq.  layout "interleaved" pairs
    values (2i, 2i + 1), "half" (i, i + rotary_dim / 2); base, scaling, factor and
    original_length as for cuda_ops.rotary_frequencies.

    forward(x, positions=0): x [B, T, heads, head_dim] or [rows, heads, head_dim],
    positions the first token's position or an integer array [T] or [B, T]
    ([rows] for a 3-D x).  The first call on a device copies inv_freq there, so
    it comes before a capture, as does one after inv_freq was changed."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, *,
                 layout: str = "interleaved", scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: Optional[int] = None):
        super().__init__()
        ops = _cuda_ops()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ops.ROTARY_LAYOUTS:
            raise ValueError(f"layout must be one of {ops.ROTARY_LAYOUTS}, got {layout!r}")
        if rotary_dim > head_dim:
            raise ValueError(f"rotary_dim ({rotary_dim}) exceeds head_dim ({head_dim})")
        self.head_dim = head_dim
        self.layout = layout
        self.inv_freq, self.scale = ops.rotary_frequencies(rotary_dim, base, scaling=scaling, factor=factor,
                                                           original_length=original_length)
        self._on = {}  # (inv_freq, its version, its copy) for each device it was used on

    def _frequencies_on(self, device):
        """inv_freq's copy on a device.  New frequencies of the same number go into
        the same memory, so steps captured before turn by them as well."""
        import torch

        src = self.inv_freq
        # tensors made in inference mode count no versions: their values stand for one
        version = src.tolist() if src.is_inference() else src._version
        kept = self._on.get(device)
        if kept is None or kept[0] is not src or kept[1] != version:
            with torch.inference_mode(False):
                if kept is not None and kept[2].shape == src.shape and kept[2].dtype == src.dtype:
                    copy = kept[2].copy_(src)
                else:
                    copy = src.to(device, copy=True)
                self._on[device] = (src, version, copy)
            return copy
        return kept[2]

    def turn(self, x, positions=0, inplace: bool = False):
        """The CUDA form on torch tensors (af_rotary)."""
        import torch

        if not isinstance(positions, (int, np.integer)):
            if not isinstance(positions, torch.Tensor):
                positions = torch.as_tensor(np.asarray(positions))
            positions = positions.to(x.device)
        return _cuda_ops().rotary(x, self._frequencies_on(x.device), positions, layout=self.layout, scale=self.scale, inplace=inplace)

    def turn_numpy(self, x: np.ndarray, positions=0) -> np.ndarray:
        """The same formula on the host, angles in 64 bits; positions as for turn."""
        if isinstance(positions, (int, np.integer)):
            positions = int(positions) + np.arange(x.shape[-3])
        positions = np.asarray(positions)
        if positions.dtype not in (np.int32, np.int64):
            raise ValueError(f"positions: expected int32 or int64, got {positions.dtype}")
        if positions.shape not in (x.shape[-3:-2], x.shape[:-2]):
            raise ValueError(f"positions of shape {positions.shape} do not match x {x.shape}")
        th = np.asarray(positions, np.float64)[..., None, None] * self.inv_freq.numpy().astype(np.float64)
        cos, sin = (self.scale * f(th) for f in (np.cos, np.sin))
        half = self.inv_freq.numel()
        if self.layout == "interleaved":
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            first, second = slice(0, half), slice(half, 2 * half)
        a, b = x[..., first], x[..., second]
        out = x.copy()
        out[..., first] = a * cos - b * sin
        out[..., second] = a * sin + b * cos
        return out

    def forward(self, x: Tensor, positions=0) -> Tensor:
        if x.shape[-1] != self.head_dim:
            raise ValueError(f"heads of {x.shape[-1]} values, expected {self.head_dim}")
        if x.device.is_cuda:
            return Tensor._wrap(self.turn(x.torch, positions), x.device)
        return Tensor(self.turn_numpy(x.numpy(), positions), x.device)


class LayerNorm(Module):
    """Standard LayerNorm (layers.py:52-67).  Not on the retention path:
    kept for API completeness on CPU tensors only."""

    def __init__(self, d_model: int, eps: float = 1e-5):
        super().__init__()
        self.d_model = d_model
        self.eps = eps
        self.weight = Parameter(Tensor(np.ones(d_model, dtype=np.float32)))
        self.bias = Parameter(Tensor(np.zeros(d_model, dtype=np.float32)))

    def forward(self, x: Tensor) -> Tensor:
        if x.device.is_cuda:
            raise NotImplementedError("LayerNorm is not part of the retention hot path (no CUDA kernel)")
        arr = x.numpy()
        mean = np.mean(arr, axis=-1, keepdims=True)
        var = np.var(arr, axis=-1, keepdims=True)
        return Tensor(((arr - mean) / np.sqrt(var + self.eps)) * self.weight.numpy() + self.bias.numpy(), x.device)


class SwiGLU(Module):
    """SwiGLU feed-forward network (layers.py:70-88): W_down(silu(W_gate x) * W_up x).

    On CUDA the gate and up weights are packed into one [2f, d] matrix (gate
    rows first, the layout of AceEngine's w_gate_up, cpu/swiglu.rs:7-8), so
    the pair is one GEMM followed by the fused SwiGLU kernel.
    """

    def __init__(self, d_model: int, hidden_dim: Optional[int] = None, multiple_of: int = 64):
        super().__init__()
        if hidden_dim is None:
            hidden_dim = int(2 * (4 * d_model) / 3)
            hidden_dim = multiple_of * ((hidden_dim + multiple_of - 1) // multiple_of)
        self.hidden_dim = hidden_dim
        self.w_gate = Linear(d_model, hidden_dim, bias=False)
        self.w_up = Linear(d_model, hidden_dim, bias=False)
        self.w_down = Linear(hidden_dim, d_model, bias=False)
        self._gate_up = None

    def _on_device(self) -> None:
        self._gate_up = None
        if self.w_gate.weight.device.is_cuda:
            import torch

            self._gate_up = torch.cat([self.w_gate.weight.torch, self.w_up.weight.torch], 0).contiguous()

    def forward(self, x: Tensor) -> Tensor:
        if x.device.is_cuda:
            ops = _cuda_ops()
            if self._gate_up is None:
                self._on_device()
            if self._gate_up is None:
                raise ValueError("SwiGLU weights are not on the input's CUDA device; call .to(device) first")
            gu = ops.linear(x.torch, self._gate_up)
            h = ops.swiglu_packed(gu)
            return Tensor._wrap(ops.linear(h, self.w_down.weight.torch), x.device)
        gate = self.w_gate(x).numpy()
        up = self.w_up(x).numpy()
        silu = gate / (1.0 + np.exp(-gate))
        return self.w_down(Tensor(silu * up, x.device))
