"""The residual-norm seam (af_residual_norm and its backward) at gates far from
zero and in views, where its precision and its strides go wrong first."""
import numpy as np
import pytest
import torch

from oracle import layer_ops_ref as L

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("d", [40, 1000, 1531, 4100, 8192, 9001])
@pytest.mark.parametrize("ht", [F32, BF16])
def test_gates_far_from_zero_in_fp32(dev, d, ht):
    """z = swish(gate) where x is 0 and h 1.  CUDA's expf is off by at most 2 units
    (2 * 2^-23), the sum, the division and the product by half a one each (2^-24): below
    2^-22 + 3 * 2^-24 of the value."""
    from aceflow_b200 import cuda_ops

    g = torch.linspace(-80.0, 20.0, 7 * d, device=dev).view(7, d).to(ht)
    x, h = torch.zeros(7, d, device=dev), torch.ones(7, d, device=dev, dtype=ht)
    z, _ = cuda_ops.residual_norm(x, h, gate=g)
    ref = L.swish64(g.double().cpu().numpy())
    assert np.all(np.abs(z.double().cpu().numpy() - ref) <= (2.0 ** -22 + 3 * 2.0 ** -24) * np.abs(ref) * 1.01)


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, mag, rel, name):
    step = 1.01 * 2.0 ** -8 * np.abs(ref) if got.dtype == BF16 else 0.0
    err = np.abs(_np(got).reshape(ref.shape) - ref)
    assert np.all(err <= rel * mag + step + 1e-37), name


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("off,width,gap", [(0, 40, 64), (1, 41, 64), (8, 64, 64), (3, 1531, 8), (8, 1531, 8), (0, 4104, 24),
                                           (5, 9000, 1)])
def test_every_result_of_views(dev, off, width, gap, dt):
    """Three-dimensional views of wider buffers, with offsets that force single
    values: both outputs, the statistics and all six gradients.  The bounds are
    100 * 2^-24 of a result's terms, and 1e-5 of a column sum's (three statistics and
    some 15 roundings a value; 24 rows)."""
    from aceflow_b200 import cuda_ops

    g = torch.Generator(device=dev).manual_seed(width)
    x, h, gate, dz, dy = (torch.randn(4, 6, off + width + gap, generator=g, device=dev).to(dt)[..., off:off + width]
                          for _ in range(5))
    w = {k: 0.5 + torch.rand(width, generator=g, device=dev) for k in ("post_w", "scale", "pre_w")}
    before = [t.clone() for t in (x, h, gate, dz, dy)]
    z, y, stats = cuda_ops.residual_norm(x, h, gate=gate, alpha=1.3, want_stats=True, **w)
    grads = cuda_ops.residual_norm_backward(dz, dy, x, h, stats, gate=gate, alpha=1.3, **w)
    assert all(torch.equal(a, b) for a, b in zip(before, (x, h, gate, dz, dy)))
    flat = lambda t: _np(t).reshape(24, width)  # noqa: E731
    ref, mag = L.seam64(flat(x), flat(h), flat(gate), alpha=1.3, dz=flat(dz), dy=flat(dy), grads=True,
                        **{k: _np(v) for k, v in w.items()})
    assert z.shape == y.shape == x.shape and z.is_contiguous() and y.is_contiguous()
    _close(z, ref["z"], mag["z"], 6e-6, "z")
    _close(y, ref["y"], mag["y"], 6e-6, "y")
    r1 = 1.0 / np.sqrt(np.square(flat(h)).mean(-1) + 1e-6)
    r2 = 1.0 / np.sqrt(np.square(ref["z"]).mean(-1) + 1e-6)
    assert np.allclose(_np(stats), np.stack([r1, r2]), rtol=6e-6, atol=0)
    for name in ("x", "h", "gate"):
        _close(getattr(grads, name), ref[name], mag[name], 6e-6, "d" + name)
    for name in ("post_w", "scale", "pre_w"):
        _close(getattr(grads, name), ref[name], mag[name], 1e-5, "d" + name)


def test_a_second_derivative_raises(dev):
    from aceflow_b200 import cuda_ops

    x, h = (torch.randn(3, 64, device=dev, requires_grad=True) for _ in range(2))
    z, y = cuda_ops.residual_norm_autograd(x, h, pre_w=torch.ones(64, device=dev))
    gx, gh = torch.autograd.grad(z.sum() + y.sum(), (x, h), create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(gx.square().sum() + h.sum(), (x, h))
    z, y = cuda_ops.residual_norm_autograd(x, h, pre_w=torch.ones(64, device=dev))
    again, _ = torch.autograd.grad(z.sum() + y.sum(), (x, h))
    assert torch.equal(again, gx) and not again.requires_grad
