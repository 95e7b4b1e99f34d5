"""What needs no GPU of the operators around the retention core, where it goes
wrong first: second derivatives (of stand-ins for the device calls), in-place
turns of tensors that autograd needs, settings and positions out of range."""
import numpy as np
import pytest
import torch

from aceflow_b200 import cuda_ops


def _turn(x, f, positions=0, *, layout="half", scale=1.0, inverse=False, inplace=False):
    th = torch.as_tensor(positions + torch.arange(x.shape[-3]))[:, None, None] * f
    c, s = scale * th.cos(), scale * (-th.sin() if inverse else th.sin())
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1).detach()


def test_second_derivative_of_the_rotation(monkeypatch):
    """|gradient|^2 as a penalty, against the same through torch's own operations."""
    monkeypatch.setattr(cuda_ops, "rotary", _turn)
    f = torch.tensor([0.5, 0.1])
    got = []
    for own in (True, False):
        x = torch.linspace(-1, 2, 24).view(1, 3, 2, 4).requires_grad_()
        if own:
            y = cuda_ops.rotary_autograd(x, f, 3, layout="half", scale=1.5)
        else:
            th = (3 + torch.arange(3))[:, None, None] * f
            a, b = x.chunk(2, -1)
            y = 1.5 * torch.cat((a * th.cos() - b * th.sin(), a * th.sin() + b * th.cos()), -1)
        g, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
        assert g.requires_grad
        got.append(torch.autograd.grad(g.square().sum() + x.sum(), x)[0])
    assert torch.allclose(got[0], got[1], rtol=1e-4, atol=1e-4)


def _seam(*args, want_stats=False, out_dtype=None, **kw):
    return args[0] * 2, args[0] * 3, torch.zeros(2, args[0].shape[0])


def _seam_grads(dz, dy, x, h, stats, *, gate, post_w, scale, pre_w, alpha):
    like = [None if t is None else torch.ones_like(t) for t in (x, h, gate, post_w, scale, pre_w)]
    return cuda_ops.ResidualNormGrads(*like)


@pytest.mark.parametrize("linear", [True, False])
def test_second_derivative_of_the_seam_raises(monkeypatch, linear):
    """Also where the loss is linear in the outputs, so that the upstream gradient
    is a constant: the seam's gradients depend on x all the same."""
    monkeypatch.setattr(cuda_ops, "residual_norm", _seam)
    monkeypatch.setattr(cuda_ops, "residual_norm_backward", _seam_grads)
    x, h, w = torch.ones(3, 4).requires_grad_(), torch.ones(3, 4), torch.ones(4).requires_grad_()
    z, y = cuda_ops.residual_norm_autograd(x, h, pre_w=w)
    loss = z.sum() + y.sum() if linear else (z * y).sum()
    gx, gw = torch.autograd.grad(loss, (x, w), create_graph=True)
    with pytest.raises(RuntimeError, match="residual_norm has no second derivative"):
        torch.autograd.grad(gx.square().sum() + x.square().sum(), x)
    loss = cuda_ops.residual_norm_autograd(x, h, pre_w=w)[0].sum()
    loss.backward()  # without create_graph nothing changes
    assert x.grad is not None and not x.grad.requires_grad and torch.all(x.grad == 1)


def test_second_derivative_of_the_retention_core_raises(monkeypatch):
    monkeypatch.setattr(cuda_ops, "retention_chunkwise_bf16", lambda qkv, *a, **k: (qkv[:, :4] * 1, None, None))
    monkeypatch.setattr(cuda_ops, "retention_chunkwise_backward_bf16", lambda qkv, *a: (torch.ones_like(qkv), None))
    qkv = torch.ones(3, 12, dtype=torch.bfloat16).requires_grad_()
    g, = torch.autograd.grad(cuda_ops.retention_chunkwise_autograd(qkv, 1, 3, 1, torch.ones(1)).sum(), qkv,
                             create_graph=True)
    with pytest.raises(RuntimeError, match="retention_chunkwise has no second derivative"):
        torch.autograd.grad(g.sum() + qkv.sum(), qkv)


def test_turning_in_place_what_autograd_needs(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_dev", lambda t: 0)
    monkeypatch.setattr(cuda_ops, "_device_call", lambda *a: None)
    f = torch.ones(2)
    x = torch.ones(1, 3, 2, 4)
    w = torch.ones_like(x).requires_grad_()
    loss = (w * x).sum()  # the product keeps x
    assert cuda_ops.rotary(x, f, inplace=True) is x
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(ValueError, match="inplace: x requires a gradient"):
        cuda_ops.rotary(w, f, inplace=True)
    with pytest.raises(ValueError, match="inplace: x requires a gradient"):
        cuda_ops.rotary((w * 2)[:, 1:], f, inplace=True)
    with torch.no_grad():
        assert cuda_ops.rotary(w, f, inplace=True) is w
    with torch.inference_mode():
        cuda_ops.rotary(torch.ones(1, 3, 2, 4), f, inplace=True)


def _given_frequencies(monkeypatch):
    """nn.Rotary.turn returns the frequencies that it hands to the device call."""
    monkeypatch.setattr(cuda_ops, "rotary", lambda x, f, *a, **k: f)


def test_rotary_module_made_in_inference_mode(monkeypatch):
    import aceflow_b200 as af

    _given_frequencies(monkeypatch)
    with torch.inference_mode():
        rot = af.nn.Rotary(8)
        x = torch.zeros(1, 2, 1, 8)
        assert torch.equal(rot.turn(x), rot.inv_freq)
    assert torch.equal(rot.turn(x), rot.inv_freq)
    with torch.inference_mode():
        rot.inv_freq *= 0.5
        assert torch.equal(rot.turn(x), rot.inv_freq)
        rot.inv_freq = rot.inv_freq * 3
    assert torch.equal(rot.turn(x), rot.inv_freq)


def test_new_frequencies_reach_captured_steps(monkeypatch):
    """They go where a captured step reads them; the tensor they replace stays."""
    import aceflow_b200 as af

    _given_frequencies(monkeypatch)
    rot, x = af.nn.Rotary(8), torch.zeros(1, 2, 1, 8)
    first = rot.inv_freq
    read = rot.turn(x)
    for change in (lambda f: f * 0.5, lambda f: f.mul_(3), lambda f: f.clone()):
        rot.inv_freq = change(rot.inv_freq)
        again = rot.turn(x)
        assert again.data_ptr() == read.data_ptr() and torch.equal(read, rot.inv_freq)
    assert first[0] == 1.0
    rot.inv_freq = torch.ones(2)
    assert rot.turn(x).tolist() == [1.0, 1.0] and read.numel() == 4


@pytest.mark.parametrize("bad", [1.5, np.array([0.0, 1.0, 2.0]), np.array(3), np.arange(2), np.zeros((3, 2), int),
                                 np.zeros((1, 3), int), np.zeros(3, np.int16), None])
def test_positions_that_the_device_refuses_are_refused_on_the_host(bad):
    import aceflow_b200 as af

    x = af.Tensor(np.ones((2, 3, 4, 8)))
    with pytest.raises(ValueError, match="positions"):
        af.nn.Rotary(8)(x, bad)
    m = af.nn.MultiScaleRetention(32, 4, rotary=af.nn.Rotary(8))
    for call in (lambda: m(af.Tensor(np.ones((2, 3, 32))), bad),
                 lambda: m.forward_chunkwise(af.Tensor(np.ones((2, 3, 32))), position=bad if bad is not None else 0.5),
                 lambda: m.forward_recurrent(af.Tensor(np.ones((3, 32))), None,
                                             bad if bad is not None and np.shape(bad) != (3,) else np.ones(3))):
        with pytest.raises(ValueError, match="positions"):
            call()


def test_positions_on_the_host():
    import aceflow_b200 as af

    rng = np.random.default_rng(1)
    rot = af.nn.Rotary(8)
    x = rng.standard_normal((2, 3, 4, 8)).astype(np.float32)
    want = rot(af.Tensor(x), 4).numpy()
    for same in (np.arange(4, 7), np.arange(4, 7, dtype=np.int32), np.tile(np.arange(4, 7), (2, 1)), np.int64(4),
                 torch.arange(4, 7)):
        assert np.array_equal(rot(af.Tensor(x), same).numpy(), want)
    m = af.nn.MultiScaleRetention(32, 4, rotary=rot)
    t = rng.standard_normal((3, 32)).astype(np.float32)
    a, _ = m.forward_recurrent(af.Tensor(t), None, 5)
    b, _ = m.forward_recurrent(af.Tensor(t), None, np.array([5, 5, 5]))
    assert np.array_equal(a.numpy(), b.numpy())


def test_top_k_beyond_31_bits_cuts_nothing(monkeypatch):
    from types import SimpleNamespace

    from aceflow_b200.engine import AceEngine

    for k, means in ((2 ** 32 + 5, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (-2 ** 32 + 5, -2 ** 31), (7, 7), (0, 0)):
        calls = []
        monkeypatch.setattr(cuda_ops, "_dev", lambda t: 0)
        monkeypatch.setattr(cuda_ops, "_ctx", lambda t: 0)
        monkeypatch.setattr(cuda_ops, "_stream", lambda t: 0)
        monkeypatch.setattr(cuda_ops, "_device_call", lambda name, *a: calls.append(a))
        monkeypatch.setattr(cuda_ops._lib, "call", lambda name, *a: calls.append(a))
        cuda_ops.sample_tokens(torch.zeros(2, 5), torch.zeros(2), top_k=k)
        cuda_ops.sample_rows(torch.zeros(2, 5), torch.zeros(2), top_k=k, temperature=1.0)
        for call in calls:
            assert means in call and (k in call) == (k == means)
        engine = SimpleNamespace(batch=2, vocab_size=5, device="cpu")
        got = AceEngine._filters(engine, 1.0, k, 1.0, 0.1, 1.0)["top_k"]
        assert got == means
        got = AceEngine._filters(engine, 1.0, [k, 3], 1.0, 0.0, 1.0)["top_k"]
        assert got.dtype == torch.int32 and got.tolist() == [means, 3]


def test_settings_of_any_kind_reach_generation():
    """generate_batch's settings as it takes them before it looks at the device."""
    from types import SimpleNamespace

    from aceflow_b200.engine import AceEngine

    class Reached(Exception):
        pass

    def stop(*settings):
        raise Reached(settings)

    engine = SimpleNamespace(_check_generate=lambda: None, _filters=stop, batch=2, vocab_size=5, device="cpu")
    engine._setting = getattr(AceEngine, "_setting", None)
    for t in (torch.tensor(0.5, dtype=torch.bfloat16), torch.tensor([0.5, 0.5]).bfloat16(), [0.5, 0.5], 0.5,
              np.float32(0.5)):
        with pytest.raises(Reached) as e:
            AceEngine.generate_batch(engine, [[1], [1]], 1, temperature=t, top_k=torch.tensor([1, 2]), top_p=0.5)
        t, k, p, m, r = (np.asarray(v) for v in e.value.args[0])
        assert np.all(t == 0.5) and k.tolist() == [1, 2] and p == 0.5 and m == 0.0 and r == 1.0
    got = AceEngine._filters(engine, np.asarray([[0.5], [1.0]]), np.asarray([[3], [2 ** 40]]), np.asarray(0.9), 0.1, 1.0)
    assert got["temperature"].tolist() == [0.5, 1.0] and got["top_k"].tolist() == [3, 2 ** 31 - 1]
    assert got["top_p"] == 0.9 and got["min_p"] == 0.1


def test_gradients_with_a_graph_may_be_changed_in_place(monkeypatch):
    monkeypatch.setattr(cuda_ops, "residual_norm", _seam)
    monkeypatch.setattr(cuda_ops, "residual_norm_backward", _seam_grads)
    x, h, w = (torch.ones(3, 4, requires_grad=True), torch.ones(3, 4, requires_grad=True),
               torch.ones(4, requires_grad=True))
    z, y = cuda_ops.residual_norm_autograd(x, h, pre_w=w)
    for g in torch.autograd.grad((z * y).sum(), (x, h, w), create_graph=True):
        assert g.requires_grad
        g.mul_(2.0)
        assert torch.all(g == 2)
    z, y = cuda_ops.residual_norm_autograd(x, h, pre_w=w)
    (z * y).sum().backward(create_graph=True)
    opt = torch.optim.SGD([x, h, w], lr=0.1)
    opt.zero_grad(set_to_none=False)
    assert torch.all(x.grad == 0) and not x.grad.requires_grad
