"""The residual-norm seam (af_residual_norm and its backward) against a
float64 evaluation.

Tolerance: each fp32 output is a sum of a few products; its rounding errors
are relative to the sum of its terms' absolute values (``mag`` of the
oracle).  A row's sums go over at most 32 values per thread and a tree of 10
levels, so a statistic is off by at most 21 units of 2^-24 after the square
root, a gradient takes three statistics and about 15 roundings: below
100 * 2^-24 = 6e-6.  A column sum of R rows adds at most 48 + 8 roundings of
2^-24 per term for the sizes here (rows per block, then parts): 1e-5.  bf16
outputs add half a step, 2^-8 of the value.
"""
import itertools

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


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _close(got, ref, mag, rel, name):
    step = 1.01 * 2.0 ** -8 * np.abs(ref) if got.dtype == BF16 else 0.0
    err = np.abs(_np(got).reshape(ref.shape) - ref)
    tol = rel * mag + step + 1e-37
    assert np.all(err <= tol), (name, float(np.max(err / tol)))


def _case(dev, rows, d, xt, ht, yt, gate, post, scale, pre, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + rows * 31 + d)
    r = lambda dt, s=1.0: (s * torch.randn(rows, d, generator=g, device=dev)).to(dt)  # noqa: E731
    w = lambda on, m: m + 0.1 * torch.randn(d, generator=g, device=dev) if on else None  # noqa: E731
    t = dict(x=r(xt, 2.0), h=r(ht, 0.7), gate=r(ht, 1.5) if gate else None, post_w=w(post, 1.0),
             scale=w(scale, 0.3), pre_w=w(pre, 1.0))
    return t, r(xt, 0.5), r(yt, 0.5) if pre else None


def _check(t, dz, dy, yt, alpha, eps=1e-6):
    from aceflow_b200 import cuda_ops

    kw = {k: t[k] for k in ("gate", "post_w", "scale", "pre_w")}
    z, y, stats = cuda_ops.residual_norm(t["x"], t["h"], alpha=alpha, eps=eps, out_dtype=yt, want_stats=True, **kw)
    g = cuda_ops.residual_norm_backward(dz, dy, t["x"], t["h"], stats, alpha=alpha, **kw)
    ref, mag = L.seam64(**{k: _np(v) for k, v in t.items()}, alpha=alpha, eps=eps, dz=_np(dz), dy=_np(dy), grads=True)
    assert z.dtype == t["x"].dtype and (y is None) == (t["pre_w"] is None)
    _close(z, ref["z"], mag["z"], 6e-6, "z")
    if y is not None:
        assert y.dtype == yt
        _close(y, ref["y"], mag["y"], 6e-6, "y")
    for name in ("x", "h", "gate"):
        got = getattr(g, name)
        assert (got is None) == (t[name] is None)
        if got is not None:
            assert got.dtype == t[name].dtype
            _close(got, ref[name], mag[name], 6e-6, "d" + name)
    for name in ("post_w", "scale", "pre_w"):
        got = getattr(g, name)
        assert (got is None) == (t[name] is None)
        if got is not None:
            _close(got, ref[name], mag[name], 1e-5, "d" + name)
    return z, y, g


@pytest.mark.parametrize("gate,post,scale,pre", list(itertools.product([False, True], repeat=4)))
def test_every_combination_of_parts(dev, gate, post, scale, pre):
    t, dz, dy = _case(dev, 5, 520, F32, F32, F32, gate, post, scale, pre)
    _check(t, dz, dy, F32, 1.3)


@pytest.mark.parametrize("xt,ht,yt", list(itertools.product([F32, BF16], repeat=3)))
@pytest.mark.parametrize("d", [256, 203])
def test_types(dev, xt, ht, yt, d):
    t, dz, dy = _case(dev, 9, d, xt, ht, yt, True, True, True, True)
    _check(t, dz, dy, yt, 1.0)


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 8), (7, 64), (130, 264), (4, 512), (6, 1000), (700, 1016),
                                    (5, 2048), (3, 4096), (2, 4104), (3, 8192), (2, 16384), (2, 127), (2, 129),
                                    (3, 513), (2, 1025), (2, 2049), (2, 4097), (2, 8191), (2, 8193), (2, 16383)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_widths(dev, rows, d, dt):
    t, dz, dy = _case(dev, rows, d, dt, dt, dt, True, True, True, True)
    _check(t, dz, dy, dt, 0.7)


def test_many_rows_share_the_column_sums_and_repeat_bit_for_bit(dev):
    t, dz, dy = _case(dev, 3001, 96, BF16, BF16, BF16, True, True, True, True)
    a = _check(t, dz, dy, BF16, 1.0)
    b = _check(t, dz, dy, BF16, 1.0)
    for p, q in zip(a[2], b[2]):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_views_with_row_strides_and_odd_offsets(dev, dt):
    """Rows inside wider buffers, an odd storage offset, three dimensions."""
    for off, width in ((0, 40), (1, 41), (8, 64)):
        big = [torch.randn(4, 6, width + 64 + off, device=dev).to(dt)[..., off:off + width] for _ in range(5)]
        t = dict(x=big[0], h=big[1], gate=big[2], post_w=torch.rand(width, device=dev) + 0.5,
                 scale=torch.rand(width, device=dev), pre_w=torch.rand(width, device=dev) + 0.5)
        from aceflow_b200 import cuda_ops

        kw = {k: t[k] for k in ("gate", "post_w", "scale", "pre_w")}
        z, y, st = cuda_ops.residual_norm(t["x"], t["h"], want_stats=True, **kw)
        flat = {k: v.reshape(24, width).contiguous() if v.dim() == 3 else v for k, v in t.items()}
        fkw = {k: flat[k] for k in ("gate", "post_w", "scale", "pre_w")}
        z2, y2, st2 = cuda_ops.residual_norm(flat["x"], flat["h"], want_stats=True, **fkw)
        assert z.shape == (4, 6, width)
        ref, mag = L.seam64(**{k: _np(v) for k, v in flat.items()})
        _close(z, ref["z"].reshape(4, 6, width), mag["z"].reshape(4, 6, width), 6e-6, "z")
        _close(y2, ref["y"], mag["y"], 6e-6, "y")
        g = cuda_ops.residual_norm_backward(big[3], big[4], t["x"], t["h"], st, **kw)
        ref, mag = L.seam64(**{k: _np(v) for k, v in flat.items()}, dz=_np(big[3]).reshape(24, width),
                            dy=_np(big[4]).reshape(24, width), grads=True)
        _close(g.h, ref["h"].reshape(4, 6, width), mag["h"].reshape(4, 6, width), 6e-6, "dh")
        _close(g.post_w, ref["post_w"], mag["post_w"], 1e-5, "dpost_w")


def test_missing_upstream_gradients_and_no_rows(dev):
    t, dz, dy = _case(dev, 6, 72, F32, F32, F32, True, True, True, True)
    _check(t, None, dy, F32, 1.1)
    _check(t, dz, None, F32, 1.1)
    _check(t, None, None, F32, 1.1)
    t, dz, dy = _case(dev, 0, 72, F32, BF16, BF16, True, True, True, True)
    z, y, g = _check(t, dz, dy, BF16, 1.0)
    assert z.shape == (0, 72) and torch.all(g.pre_w == 0) and torch.all(g.scale == 0)


def test_zero_rows_closed_gates_and_extremes(dev):
    """A row of zeros has finite norms; a gate of the type's lowest value or
    -inf closes; large values do not overflow where the formula does not."""
    from aceflow_b200 import cuda_ops

    d = 64
    x, h = torch.zeros(4, d, device=dev), torch.zeros(4, d, device=dev)
    h[1:] = torch.randn(3, d, device=dev)
    x[2] = 1e15
    gate = torch.randn(4, d, device=dev)
    gate[3, ::2] = float("-inf")
    gate[3, 1::2] = torch.finfo(F32).min
    w = torch.ones(d, device=dev)
    z, y, st = cuda_ops.residual_norm(x, h, gate=gate, post_w=w, scale=w, pre_w=w, want_stats=True)
    assert torch.isfinite(z).all() and torch.isfinite(y).all()
    assert torch.all(z[0] == 0) and torch.all(y[0] == 0) and torch.all(z[3] == 0)
    assert torch.allclose(y[2], torch.ones_like(y[2]))
    g = cuda_ops.residual_norm_backward(torch.ones_like(z), torch.ones_like(y), x, h, st, gate=gate, post_w=w, scale=w,
                                        pre_w=w)
    for v in g:
        assert torch.isfinite(v).all()
    assert torch.all(g.gate[3] == 0) and torch.all(g.h[3] == 0)


def test_autograd_and_a_shared_input(dev):
    """Gradients through torch: x used twice, an output that the loss leaves
    out, an expanded upstream gradient; against the direct call."""
    from aceflow_b200 import cuda_ops

    t, dz, dy = _case(dev, 6, 80, F32, F32, F32, True, True, True, True)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    kw = {k: leaves[k] for k in ("gate", "post_w", "scale", "pre_w")}
    z, y = cuda_ops.residual_norm_autograd(leaves["x"], leaves["h"], alpha=1.2, **kw)
    ((z * dz).sum() + (y * dy).sum() + leaves["x"].sum()).backward()
    ref, mag = L.seam64(**{k: _np(v) for k, v in t.items()}, alpha=1.2, dz=_np(dz), dy=_np(dy), grads=True)
    ref["x"] += 1.0
    mag["x"] += 1.0
    for k in leaves:
        _close(leaves[k].grad, ref[k], mag[k], 1e-5, k)
    x = t["x"].clone().requires_grad_()
    z, y = cuda_ops.residual_norm_autograd(x, t["h"], pre_w=t["pre_w"])
    y.sum().backward()
    ref, mag = L.seam64(_np(t["x"]), _np(t["h"]), pre_w=_np(t["pre_w"]), dy=np.ones((6, 80)), grads=True)
    _close(x.grad, ref["x"], mag["x"], 6e-6, "x")
    same = t["h"].clone().requires_grad_()
    z, y = cuda_ops.residual_norm_autograd(same, same, pre_w=t["pre_w"])
    z.sum().backward()
    assert torch.allclose(same.grad, torch.full_like(same, 2.0))


def test_two_graphs_and_another_stream(dev):
    """Forward and backward captured into two graphs of different sizes and
    replayed in turn; each keeps its own scratch."""
    from aceflow_b200 import cuda_ops

    sets = [_case(dev, r, 128, F32, BF16, BF16, True, True, True, True) for r in (40, 900)]

    def step(t, dz, dy):
        kw = {k: t[k] for k in ("gate", "post_w", "scale", "pre_w")}
        z, y, st = cuda_ops.residual_norm(t["x"], t["h"], want_stats=True, **kw)
        return (z, y) + tuple(cuda_ops.residual_norm_backward(dz, dy, t["x"], t["h"], st, **kw))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = [[v.clone() for v in step(*c)] for c in sets]
    s.synchronize()
    graphs, outs = [], []
    for c in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*c))
        graphs.append(g)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for a, b in zip(w, o):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,d", [(9, 1), (40, 3), (33, 7), (2500, 9), (17, 130), (2400, 241), (1300, 249), (11, 250),
                                    (1021, 1531), (700, 2030), (310, 4089), (5, 4090), (160, 5003), (3, 8185), (3, 8186)])
@pytest.mark.parametrize("xt,ht", [(F32, F32), (BF16, BF16), (F32, BF16)])
def test_rows_that_start_anywhere(dev, rows, d, xt, ht):
    """Widths that are no multiple of 8: rows start anywhere in 16 bytes, a
    thread's vectors reach into the rows next to its own, groups of rows walk."""
    t, dz, dy = _case(dev, rows, d, xt, ht, ht, True, True, True, True)
    _check(t, dz, dy, ht, 1.2)


@pytest.mark.parametrize("d,gap", [(1531, 8), (1531, 3), (75, 16), (5003, 8), (512, 8), (512, 3)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_what_lies_between_rows_does_not_matter(dev, d, gap, dt):
    """NaN between the rows of every input, and rows before and behind."""
    rows = 400
    t, dz, dy = _case(dev, rows, d, dt, dt, dt, True, True, True, True)

    def inside(v):
        big = torch.full((rows + 2, d + gap), float("nan"), device=dev, dtype=dt)
        skip = 8 * ((d + gap) // 8 + 1) if (d + gap) % 8 else d + gap  # the first row starts on 16 bytes
        view = big.view(-1)[skip:].as_strided((rows, d), (d + gap, 1))
        view.copy_(v)
        return view

    for k in ("x", "h", "gate"):
        t[k] = inside(t[k])
    _check(t, inside(dz), inside(dy), dt, 0.9)


def test_more_rows_than_counters_hold_are_refused(dev):
    from aceflow_b200 import cuda_ops

    assert cuda_ops._seam_scratch(0, 2**30, 8) > 0
    with pytest.raises(ValueError, match="bad sizes"):
        cuda_ops._seam_scratch(0, 2**30 + 1, 8)


def test_offsets_beyond_31_bits(dev):
    """More than 2^31 values: the last rows are those of a small call."""
    from aceflow_b200 import cuda_ops

    rows, d, last = 1073800, 2001, 5  # rows that start anywhere
    g = torch.Generator(device=dev).manual_seed(5)
    x, h, dz = (torch.zeros(rows, d, device=dev, dtype=BF16) for _ in range(3))
    w = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
    for t in (x, h, dz):
        t[-last:] = torch.randn(last, d, generator=g, device=dev).to(BF16)
    small = [t[-last:].clone() for t in (x, h, dz)]
    z, y, stats = cuda_ops.residual_norm(x, h, post_w=w, pre_w=w, want_stats=True)
    sz, sy, sstats = cuda_ops.residual_norm(*small[:2], post_w=w, pre_w=w, want_stats=True)
    assert torch.equal(z[-last:], sz) and torch.equal(y[-last:], sy) and not z[0].any()
    del z, y
    got = cuda_ops.residual_norm_backward(dz, None, x, h, stats, post_w=w, pre_w=w)
    ref = cuda_ops.residual_norm_backward(small[2], None, *small[:2], sstats, post_w=w, pre_w=w)
    assert torch.equal(got.x[-last:], ref.x) and torch.equal(got.h[-last:], ref.h)
    # the same terms and zeros, in another grouping
    assert torch.allclose(got.post_w, ref.post_w, rtol=1e-5, atol=1e-5)
