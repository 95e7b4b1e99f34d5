"""The operators around the retention core inside the layer and the engine, in
the calls that their other tests leave out.  Tolerances are the framework's own:
fp32 1e-4, bf16 tensor-core products 2e-2 of the largest value."""
import numpy as np
import pytest
import torch

from conftest import rel_err

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("chunk", [64, 128])
def test_a_rotated_prompt_continues_from_a_state(dev, gated, chunk):
    """A prompt in three parts of odd lengths, positions as a number, per token and
    per stream, against the prompt in one."""
    import aceflow_b200 as af

    B, T, d, at = 2, 150, 512, 70000
    np.random.seed(12)
    m = af.nn.MultiScaleRetention(d, 2, gated=gated, rotary=af.nn.Rotary(256, layout="half")).to("cuda:0")
    x = torch.randn(B, T, d, generator=torch.Generator().manual_seed(3)).bfloat16().to(dev)
    part = lambda a, b: af.Tensor(x[:, a:b].contiguous(), device="cuda:0", dtype="bfloat16")  # noqa: E731
    whole, end = m.forward_chunkwise(part(0, T), chunk=chunk, position=at)
    a, st = m.forward_chunkwise(part(0, 67), chunk=chunk, position=at)
    kept = st.numpy().copy()
    b, st2 = m.forward_chunkwise(part(67, 68), chunk=chunk, state=st, position=np.array([at + 67]))
    c, st3 = m.forward_chunkwise(part(68, T), chunk=chunk, state=st2,
                                 position=torch.arange(at + 68, at + T, device=dev).repeat(B, 1))
    assert np.array_equal(st.numpy(), kept)
    got = np.concatenate([v.numpy().astype(np.float32) for v in (a, b, c)], 1)
    assert rel_err(got, whole.numpy().astype(np.float32)) < 2e-2 and rel_err(st3.numpy(), end.numpy()) < 2e-2
    wrong, _ = m.forward_chunkwise(part(68, T), chunk=chunk, state=st2, position=0)
    assert rel_err(wrong.numpy().astype(np.float32), whole.numpy()[:, 68:].astype(np.float32)) > 2e-2


def test_generation_takes_settings_from_the_device(dev):
    from aceflow_b200.engine import AceEngine

    rng = np.random.default_rng(21)
    w = lambda *s: (0.2 * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    V, d, B, n = 300, 128, 3, 5
    e = AceEngine(1, d, 2, w(V, d), batch=B)
    e.load_layer_weights(0, w(3 * d, d), w(d, d), w(2 * 256, d), w(d, 256), np.ones(d), np.ones(d))
    prompts, u = rng.integers(0, V, (B, 9)), rng.random((B, n)).astype(np.float32)

    def run(**kw):
        e.reset_memory()
        return e.generate_batch(prompts, n, uniforms=u, **kw)

    t = lambda v, dt=torch.float32: torch.tensor(v, device=dev, dtype=dt)  # noqa: E731
    assert np.array_equal(run(temperature=0.75, top_k=30), run(temperature=t(0.75), top_k=t(30, torch.int64)))
    host = dict(temperature=[0.0, 0.75, 1.25], top_k=[0, 40, 2 ** 33], min_p=[0.0, 0.0625, 0.0])
    want = run(**host)
    assert np.array_equal(want, run(temperature=t(host["temperature"]).bfloat16(), top_k=t(host["top_k"], torch.int64),
                                    min_p=t(host["min_p"])))
    with pytest.raises(ValueError, match="min_p"):
        run(temperature=1.0, min_p=t([0.1, 0.1]))
