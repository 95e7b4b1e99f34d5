"""What needs no GPU of the operators around the retention core: refusals
(before any device call), the frequency helper, and the oracle's own formulas
(gradients against differences, draws worked by hand)."""
import math

import numpy as np
import pytest
import torch

from aceflow_b200 import cuda_ops
from oracle import layer_ops_ref as L


def test_frequencies():
    f, s = cuda_ops.rotary_frequencies(8, 100.0)
    assert s == 1.0 and np.allclose(f.numpy(), [1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-6)
    lin, _ = cuda_ops.rotary_frequencies(8, 100.0, scaling="linear", factor=4.0)
    assert np.allclose(lin.numpy(), f.numpy() / 4, rtol=1e-6)
    ntk, _ = cuda_ops.rotary_frequencies(8, 100.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and np.isclose(float(ntk[-1]), float(f[-1]) / 4, rtol=1e-5)
    yarn, s = cuda_ops.rotary_frequencies(64, scaling="yarn", factor=16.0, original_length=4096)
    plain, _ = cuda_ops.rotary_frequencies(64)
    ratio = yarn.double().numpy() / plain.double().numpy()
    assert np.isclose(s, 0.1 * math.log(16) + 1) and ratio[0] == 1.0 and np.isclose(ratio[-1], 1 / 16, rtol=1e-5)
    assert np.all(np.diff(ratio) <= 1e-7)
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, scaling="cubic"), dict(rot_dim=8, factor=0.0),
                dict(rot_dim=8, base=-1.0), dict(rot_dim=8, scaling="yarn", factor=2.0),
                dict(rot_dim=8, scaling="yarn", original_length=9, beta_fast=1.0)):
        with pytest.raises(ValueError):
            cuda_ops.rotary_frequencies(**bad)


@pytest.mark.parametrize("change,match", [
    (dict(x=torch.zeros(4, 8)), "x must be"), (dict(x=torch.zeros(1, 4, 2, 8).double()), "float32 or bfloat16"),
    (dict(x=torch.zeros(1, 4, 2, 16)[..., ::2]), "unit stride"), (dict(layout="pairs"), "layout"),
    (dict(f=torch.zeros(5)), "frequencies"), (dict(f=torch.zeros(0)), "frequencies"),
    (dict(f=torch.zeros(2, 2)), "frequencies"), (dict(f=torch.zeros(4, dtype=torch.float64)), "inv_freq"),
    (dict(), "CUDA")])
def test_rotary_refusals(change, match):
    a = dict(x=torch.zeros(1, 4, 2, 8), f=torch.zeros(4), layout="half") | change
    with pytest.raises(ValueError, match=match):
        cuda_ops.rotary(a["x"], a["f"], layout=a["layout"])


@pytest.mark.parametrize("change,match", [
    (dict(h=torch.zeros(3, 9)), "h: expected shape"), (dict(x=torch.zeros(3, 8).half()), "x: expected"),
    (dict(gate=torch.zeros(3, 8, dtype=torch.bfloat16)), "gate"), (dict(gate=torch.zeros(2, 8)), "gate"),
    (dict(post_w=torch.zeros(7)), "post_w"), (dict(scale=torch.zeros(8).bfloat16()), "scale"),
    (dict(pre_w=torch.zeros(16)[::2]), "pre_w"), (dict(out_dtype=torch.float16), "out_dtype"),
    (dict(x=torch.zeros(3, 0), h=torch.zeros(3, 0)), "non-empty"), (dict(), "CUDA")])
def test_residual_norm_refusals(change, match):
    a = dict(x=torch.zeros(3, 8), h=torch.zeros(3, 8)) | change
    with pytest.raises(ValueError, match=match):
        cuda_ops.residual_norm(a.pop("x"), a.pop("h"), **a)


@pytest.mark.parametrize("change,match", [
    (dict(stats=torch.zeros(3, 2)), "stats"), (dict(dz=torch.zeros(3, 8).bfloat16()), "dz"),
    (dict(dy=torch.zeros(3, 8)), "dy without pre_w"), (dict(dz=torch.zeros(8)), "dz"), (dict(), "CUDA")])
def test_residual_norm_backward_refusals(change, match):
    a = dict(dz=torch.zeros(3, 8), dy=None, stats=torch.zeros(2, 3)) | change
    with pytest.raises(ValueError, match=match):
        cuda_ops.residual_norm_backward(a["dz"], a["dy"], torch.zeros(3, 8), torch.zeros(3, 8), a["stats"])


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(2, 5).half()), "logits"), (dict(logits=torch.zeros(5)), "logits"),
    (dict(logits=torch.zeros(2, 0)), "logits"), (dict(logits=torch.zeros(5, 2).t()), "unit column stride"),
    (dict(uniforms=torch.zeros(3)), "uniforms"), (dict(uniforms=torch.zeros(2).double()), "uniforms"),
    (dict(top_k=torch.zeros(2, dtype=torch.int64)), "top_k"), (dict(top_p=torch.zeros(3)), "top_p"),
    (dict(temperature=torch.zeros(4)[::2]), "temperature"), (dict(context=torch.zeros(2, 3)), "context"),
    (dict(context=torch.zeros(3, 3, dtype=torch.int32)), "context"), (dict(repetition_penalty=0.0), "penalty"),
    (dict(), "CUDA")])
def test_sample_tokens_refusals(change, match):
    a = dict(logits=torch.zeros(2, 5), uniforms=torch.zeros(2)) | change
    with pytest.raises(ValueError, match=match):
        cuda_ops.sample_tokens(a.pop("logits"), a.pop("uniforms"), **a)


def test_oracle_seam_gradients_against_differences():
    rng = np.random.default_rng(3)
    t = dict(x=rng.standard_normal((3, 6)), h=rng.standard_normal((3, 6)), gate=rng.standard_normal((3, 6)),
             post_w=1 + 0.1 * rng.standard_normal(6), scale=rng.standard_normal(6), pre_w=rng.standard_normal(6))
    dz, dy, e = rng.standard_normal((3, 6)), rng.standard_normal((3, 6)), 1e-6
    g, _ = L.seam64(**t, alpha=1.3, dz=dz, dy=dy, grads=True)

    def loss(**c):
        v, _ = L.seam64(**(t | c), alpha=1.3)
        return float((v["z"] * dz).sum() + (v["y"] * dy).sum())

    for name, v in t.items():
        for i in np.ndindex(v.shape):
            hi, lo = v.copy(), v.copy()
            hi[i] += e
            lo[i] -= e
            assert abs((loss(**{name: hi}) - loss(**{name: lo})) / (2 * e) - g[name][i]) < 1e-6


def test_oracle_draw_worked_by_hand():
    lg = np.log(np.array([1.0, 2.0, 3.0, 4.0]))
    assert [L.sample64(lg, u)[0] for u in (0.0, 0.39, 0.41, 0.71, 0.91)] == [3, 3, 2, 1, 0]
    assert L.sample64(lg, 0.99, min_p=0.6)[0] == 2 and L.sample64(lg, 0.99, top_p=0.3)[0] == 3
    assert L.sample64([-np.inf] * 3, 0.5)[0] == -1 and L.sample64([0.0] * 5, 0.5, top_k=2)[0] == 0
    assert abs(L.sample64(lg, 0.99, min_p=0.6)[1] - math.log(3 / 7)) < 1e-6


def test_oracle_rotary_turns_back():
    rng = np.random.default_rng(4)
    x, f = rng.standard_normal((2, 5, 3, 10)), np.array([1.0, 0.3, 0.01])
    for layout in ("interleaved", "half"):
        y = L.rotary64(x, f, 7 + np.arange(5), layout, 2.0)
        assert np.allclose(L.rotary64(y, f, 7 + np.arange(5), layout, 0.5, True), x)
        assert np.array_equal(y[..., 6:], x[..., 6:])


def test_modules_on_the_cpu():
    """nn.Rotary, nn.ResidualNorm and a rotated MultiScaleRetention: the parallel
    form, the recurrence and the prompt in two parts agree."""
    import aceflow_b200 as af

    rng = np.random.default_rng(6)
    rot = af.nn.Rotary(16, 8, layout="half", scaling="linear", factor=2.0)
    x = rng.standard_normal((2, 5, 3, 16)).astype(np.float32)
    ref = L.rotary64(x, rot.inv_freq.numpy(), 3 + np.arange(5), "half")
    assert np.max(np.abs(rot(af.Tensor(x), 3).numpy() - ref)) < 1e-6
    assert list(rot.parameters()) == []
    np.random.seed(9)
    m = af.nn.MultiScaleRetention(64, 4, rotary=af.nn.Rotary(16))
    np.random.seed(9)
    assert np.array_equal(m.w_q.numpy(), af.nn.MultiScaleRetention(64, 4).w_q.numpy())
    t = rng.standard_normal((2, 9, 64)).astype(np.float32)
    full = m(af.Tensor(t), 40).numpy()
    a, st = m.forward_chunkwise(af.Tensor(t[:, :4]), position=40)
    b, st = m.forward_chunkwise(af.Tensor(t[:, 4:]), state=st, position=44)
    assert np.max(np.abs(np.concatenate([a.numpy(), b.numpy()], 1) - full)) < 1e-5
    assert np.max(np.abs(m(af.Tensor(t), 900).numpy() - full)) < 1e-4  # relative positions alone matter
    assert np.max(np.abs(m(af.Tensor(t), np.arange(9) * 3).numpy() - full)) > 1e-3
    s = af.nn.ResidualNorm(64, layer_scale=0.1)
    z, y = s(af.Tensor(t), af.Tensor(full))
    want, _ = L.seam64(t, full, None, np.ones(64), np.full(64, 0.1), np.ones(64))
    assert np.max(np.abs(z.numpy() - want["z"])) < 1e-5 and np.max(np.abs(y.numpy() - want["y"])) < 1e-5
    assert [n for n, _ in s.named_parameters()] == ["pre_weight", "post_weight", "scale"]


def test_module_refusals():
    import aceflow_b200 as af

    with pytest.raises(ValueError, match="rotary"):
        af.nn.MultiScaleRetention(64, 4, rotary=af.nn.Rotary(32))
    with pytest.raises(ValueError, match="exceeds"):
        af.nn.Rotary(16, 18)
    with pytest.raises(ValueError, match="layout"):
        af.nn.Rotary(16, layout="both")
    plain, turned = af.nn.MultiScaleRetention(64, 4), af.nn.MultiScaleRetention(64, 4, rotary=af.nn.Rotary(16))
    x = af.Tensor(np.zeros((2, 3, 64)))
    with pytest.raises(ValueError, match="position"):
        plain(x, 5)
    with pytest.raises(ValueError, match="position"):
        plain.forward_recurrent(af.Tensor(np.zeros((2, 64))), None, 5)
    with pytest.raises(ValueError, match="position"):
        turned.forward_recurrent(af.Tensor(np.zeros((2, 64))))
    with pytest.raises(ValueError, match="position"):
        turned.forward_chunkwise(x, state=turned.init_state(2))
    turned.forward_chunkwise(x, state=turned.init_state(2), position=7)
    with pytest.raises(ValueError, match="CUDA"):
        af.ops.rotary(x, af.Tensor(np.ones(4)))
