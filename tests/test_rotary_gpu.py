"""Rotary positions (af_rotary) against a float64 evaluation.

Tolerance: the angle's remainder is off by at most 2^-26 turns (1e-7 rad),
sincospif by 2 units of 2^-24, and a pair takes three more fp32 roundings:
together below 1e-6 of the pair's length.  Forming the angle in 64 bits takes
three roundings here and one in the oracle: 4 * 2^-53 of the angle, at most
the position.  A bf16 result adds half a step, 2^-8 of the value.
"""
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


def _freq(dev, rot, base=10000.0):
    from aceflow_b200 import cuda_ops

    return cuda_ops.rotary_frequencies(rot, base, device=dev)[0]


def _check(out, x, f, pos, layout, scale=1.0, inverse=False):
    ref = L.rotary64(x.double().cpu().numpy(), f.cpu().numpy(), pos, layout, scale, inverse)
    got = out.double().cpu().numpy()
    assert out.shape == x.shape and out.dtype == x.dtype
    rot = 2 * f.numel()
    xs = np.abs(x.double().cpu().numpy())
    length = np.zeros_like(ref)
    length[..., :rot] = scale * np.sqrt(2.0) * xs[..., :rot].max(-1, keepdims=True, initial=0.0)
    tol = (1e-6 + 4 * 2.0 ** -53 * np.max(np.abs(pos), initial=0.0)) * length + (2.0 ** -8 * np.abs(ref) * 1.01 if x.dtype == torch.bfloat16 else 0.0)
    tol[..., rot:] = 0.0  # the rest of a head is copied
    assert np.all(np.abs(got - ref) <= tol), float(np.max(np.abs(got - ref) - tol))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,D,rot", [(1, 1, 1, 2, 2), (2, 7, 3, 64, 64), (1, 33, 16, 256, 256), (3, 5, 2, 96, 40),
                                         (2, 9, 5, 80, 20), (1, 13, 1, 27, 26), (1, 4, 9, 33, 2), (2, 3, 4, 24, 12),
                                         (64, 1, 8, 128, 64), (1, 300, 17, 48, 34)])
def test_shapes_types_and_layouts(dev, layout, dtype, B, T, H, D, rot):
    from aceflow_b200 import cuda_ops

    g = torch.Generator(device=dev).manual_seed(B * 1000 + T * 10 + D + rot)
    x = torch.randn(B, T, H, D, generator=g, device=dev).to(dtype)
    f = _freq(dev, rot)
    out = cuda_ops.rotary(x, f, 5, layout=layout, scale=1.25)
    _check(out, x, f, np.arange(5, 5 + T), layout, 1.25)
    back = cuda_ops.rotary(x, f, 5, layout=layout, scale=1.25, inverse=True)
    _check(back, x, f, np.arange(5, 5 + T), layout, 1.25, True)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("start", [1000003, 2 ** 31 - 40, -17, 2 ** 33])
def test_far_positions_keep_their_angle(dev, layout, start):
    from aceflow_b200 import cuda_ops

    x = torch.randn(1, 20, 2, 64, device=dev)
    f = _freq(dev, 64)
    _check(cuda_ops.rotary(x, f, start, layout=layout), x, f, start + np.arange(20.0), layout)
    if abs(start) < 2 ** 31 - 20:
        pos = torch.arange(start, start + 20, device=dev, dtype=torch.int32)
        assert torch.equal(cuda_ops.rotary(x, f, pos, layout=layout), cuda_ops.rotary(x, f, start, layout=layout))
    pos = torch.arange(start, start + 20, device=dev)
    assert torch.equal(cuda_ops.rotary(x, f, pos, layout=layout), cuda_ops.rotary(x, f, start, layout=layout))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_views_of_a_packed_projection_and_in_place(dev, dtype, layout):
    """q and k inside a packed qkv, positions per stream and token (as a
    strided tensor), in place: v is left as it was."""
    from aceflow_b200 import cuda_ops

    B, T, H, D = 3, 11, 4, 64
    qkv = torch.randn(B, T, 3 * H * D, device=dev).to(dtype)
    before = qkv.clone()
    f = _freq(dev, 32)
    pos = torch.randint(0, 9000, (T, B), device=dev).t()
    qk = qkv[..., : 2 * H * D].unflatten(-1, (2 * H, D))
    out = cuda_ops.rotary(qk, f, pos, layout=layout)
    assert torch.equal(qkv, before) and out.is_contiguous()
    _check(out, qk, f, pos.cpu().numpy(), layout)
    res = cuda_ops.rotary(qk, f, pos, layout=layout, inplace=True)
    assert res.data_ptr() == qkv.data_ptr() and torch.equal(qk, out)
    assert torch.equal(qkv[..., 2 * H * D:], before[..., 2 * H * D:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_other_orders_offsets_and_expanded_inputs(dev, dtype, layout):
    from aceflow_b200 import cuda_ops

    f = _freq(dev, 16)
    heads_first = torch.randn(2, 5, 9, 32, device=dev).to(dtype).transpose(1, 2)  # [B, T, heads, dim] over [B, heads, T, dim]
    _check(cuda_ops.rotary(heads_first, f, 3, layout=layout), heads_first, f, 3 + np.arange(9), layout)
    for off in (1, 2, 4):  # every access width
        odd = torch.randn(6 * 3 * 32 + off, device=dev).to(dtype)[off:].view(1, 6, 3, 32)
        _check(cuda_ops.rotary(odd, f, layout=layout), odd, f, np.arange(6), layout)
        odd_rows = torch.randn(1, 6, 3 * 32 + off, device=dev).to(dtype)[..., : 3 * 32].unflatten(-1, (3, 32))
        _check(cuda_ops.rotary(odd_rows, f, layout=layout), odd_rows, f, np.arange(6), layout)
    one = torch.randn(1, 1, 3, 32, device=dev).to(dtype).expand(2, 4, 3, 32)
    _check(cuda_ops.rotary(one, f, layout=layout), one, f, np.arange(4), layout)
    rows = torch.randn(7, 3, 32, device=dev).to(dtype)  # 3-D: one position per row
    pos = torch.tensor([5, 0, 5, 123, 7, 7, 99], device=dev, dtype=torch.int32)
    _check(cuda_ops.rotary(rows, f, pos, layout=layout), rows, f, pos.cpu().numpy(), layout)


def test_empty_and_special_values(dev):
    from aceflow_b200 import cuda_ops

    f = _freq(dev, 8)
    for shape in ((0, 4, 2, 16), (2, 0, 2, 16), (2, 4, 0, 16), (0, 2, 16)):
        assert cuda_ops.rotary(torch.empty(shape, device=dev), f).shape == shape
    x = torch.randn(1, 3, 1, 16, device=dev)
    x[..., 8:] = float("inf")
    x[..., 9] = float("nan")
    out = cuda_ops.rotary(x, f)
    assert torch.equal(out[..., 8:].isnan(), x[..., 8:].isnan()) and torch.isfinite(out[..., :8]).all()
    assert torch.equal(out[0, 0, :, :8], x[0, 0, :, :8])  # position 0 turns nothing


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient(dev, layout):
    """Against the formula (the inverse rotation) and central differences of
    the float64 form; the gradient of an expanded result and of a view."""
    from aceflow_b200 import cuda_ops

    f, fs = cuda_ops.rotary_frequencies(12, scaling="yarn", factor=4.0, original_length=64, device=dev)
    base = torch.randn(2, 5, 3 * 16 + 16, device=dev, requires_grad=True)
    pos = torch.randint(0, 500, (2, 5), device=dev)
    x = base[..., :48].unflatten(-1, (3, 16))
    w = torch.randn(2, 5, 3, 16, device=dev)
    (cuda_ops.rotary_autograd(x, f, pos, layout=layout, scale=fs) * w).sum().backward()
    ref = L.rotary64(w.cpu().numpy(), f.cpu().numpy(), pos.cpu().numpy(), layout, fs, True)
    ref[..., 12:] = w.cpu().numpy()[..., 12:]
    got = base.grad[..., :48].unflatten(-1, (3, 16)).cpu().numpy()
    assert np.max(np.abs(got - ref)) < 2e-5 and torch.all(base.grad[..., 48:] == 0)
    xn, e = x.detach().double().cpu().numpy(), 1e-4
    for idx in [(0, 0, 0, 0), (1, 4, 2, 11), (0, 3, 1, 5), (1, 2, 0, 15)]:
        hi, lo = xn.copy(), xn.copy()
        hi[idx] += e
        lo[idx] -= e
        q = [(L.rotary64(v, f.cpu().numpy(), pos.cpu().numpy(), layout, fs) * w.cpu().numpy()).sum() for v in (hi, lo)]
        assert abs((q[0] - q[1]) / (2 * e) - got[idx]) < 1e-4
    leaf = torch.randn(2, 4, 1, 16, device=dev, requires_grad=True)
    cuda_ops.rotary_autograd(leaf, f, layout=layout).sum().backward()  # an expanded gradient arrives
    assert torch.isfinite(leaf.grad).all()


def test_decode_step_in_a_graph_with_moving_positions(dev):
    """Single tokens of streams of different lengths, captured once; the
    positions move on the device between replays."""
    from aceflow_b200 import cuda_ops

    B, H, D = 5, 6, 64
    x = torch.randn(B, H, D, device=dev)
    pos = torch.tensor([0, 3, 900, 17, 4095], device=dev, dtype=torch.int32)
    f = _freq(dev, 64)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        cuda_ops.rotary(x, f, pos)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cuda_ops.rotary(x, f, pos)
        pos += 1
    for _ in range(3):
        p = pos.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x, f, p, "interleaved")


def test_relative_positions(dev):
    """q_t . k_s of turned vectors depends on t - s alone."""
    from aceflow_b200 import cuda_ops

    q, k = torch.randn(1, 1, 1, 64, device=dev), torch.randn(1, 1, 1, 64, device=dev)
    f = _freq(dev, 64)
    dots = [float((cuda_ops.rotary(q, f, t) * cuda_ops.rotary(k, f, t - 9)).sum()) for t in (9, 1000, 123456)]
    assert max(dots) - min(dots) < 1e-6 * float(q.norm() * k.norm()) * 4
