"""Rotary positions (af_rotary) where fp32 would not do, and where an angle's
remainder is largest."""
import numpy as np
import pytest
import torch

from oracle import layer_ops_ref as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("start", [0, 32768, 10 ** 6])
def test_cosines_and_sines_to_their_last_bit(dev, layout, start):
    """Pairs (1, 0) turn into (cos, sin).  CUDA's sincospif is off by at most 2 units
    of its value (2 * 2^-23 of it), a product and a sum each by half a one (2^-24);
    the angle by 4 * 2^-53 of itself.  The remainder rounded to fp32 alone would add
    1e-7, which shows where the sine or the cosine is small."""
    from aceflow_b200 import cuda_ops

    T, D = 4096, 128
    f, _ = cuda_ops.rotary_frequencies(D, device=dev)
    x = torch.zeros(1, T, 1, D, device=dev)
    first = (slice(0, D, 2), slice(1, D, 2)) if layout == "interleaved" else (slice(0, D // 2), slice(D // 2, D))
    x[..., first[0]] = 1.0
    got = cuda_ops.rotary(x, f, start, layout=layout).double().cpu().numpy()[0, :, 0]
    th = (start + np.arange(T))[:, None] * f.double().cpu().numpy()
    for part, ref in zip(first, (np.cos(th), np.sin(th))):
        err = np.abs(got[:, part] - ref)
        # 2^-44: the second order of 1e-7, and that angle's own rounding
        assert np.all(err <= (2 * 2.0 ** -23 + 2 * 2.0 ** -24) * np.abs(ref) + 4 * 2.0 ** -53 * th + 2.0 ** -44)


def test_rounded_angles_add_no_error_on_average(dev):
    """Root mean square against 64 bits.  A rounding is off by 0.42 * 2^-24 of its
    value on average: cos and sin take one, one product of the two of a result
    (half of the square), and the sum: 0.66 together.  As much again as one
    rounding for what sincospif is off beyond it: 0.78."""
    from aceflow_b200 import cuda_ops

    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(2, 2000, 4, 128, generator=g, device=dev)
    f, _ = cuda_ops.rotary_frequencies(128, device=dev)
    got = cuda_ops.rotary(x, f, 17).double().cpu().numpy()
    ref = L.rotary64(x.double().cpu().numpy(), f.cpu().numpy(), 17 + np.arange(2000))
    assert np.linalg.norm(got - ref) <= 0.8 * 2.0 ** -24 * np.linalg.norm(ref)


def test_second_derivative(dev):
    """|gradient|^2 as a penalty, against torch's own operations in 64 bits."""
    from aceflow_b200 import cuda_ops

    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(2, 5, 3, 16, generator=g, device=dev, requires_grad=True)
    f, _ = cuda_ops.rotary_frequencies(16, 100.0, device=dev)
    y = cuda_ops.rotary_autograd(x, f, 3, layout="half", scale=1.5)
    d, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
    got, = torch.autograd.grad(d.square().sum() + x.sum(), x)
    xd = x.detach().double().requires_grad_()
    th = (3 + torch.arange(5, device=dev))[:, None, None] * f.double()
    a, b = xd.chunk(2, -1)
    y = 1.5 * torch.cat((a * th.cos() - b * th.sin(), a * th.sin() + b * th.cos()), -1)
    d, = torch.autograd.grad((y ** 3).sum(), xd, create_graph=True)
    ref, = torch.autograd.grad(d.square().sum() + xd.sum(), xd)
    # some ten roundings of a polynomial of degree 3 in y, each relative to its terms
    assert float((got - ref).abs().max()) <= 40 * 2.0 ** -24 * float(ref.abs().max())


def test_in_place_is_seen_by_autograd(dev):
    from aceflow_b200 import cuda_ops

    f, _ = cuda_ops.rotary_frequencies(8, device=dev)
    x = torch.randn(1, 3, 2, 8, device=dev)
    w = torch.ones_like(x, requires_grad=True)
    loss = (w * x).sum()
    cuda_ops.rotary(x[:, :, :1], f, inplace=True)  # a view of it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_captured_steps_turn_by_new_frequencies(dev):
    import aceflow_b200 as af

    with torch.inference_mode():
        rot = af.nn.Rotary(64)
    x = torch.randn(2, 3, 4, 64, device=dev)
    rot.turn(x, 7)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot.turn(x, 7)
    for change in (1.0, 0.25, 3.0):
        rot.inv_freq = rot.inv_freq * change
        want = rot.turn(x, 7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
