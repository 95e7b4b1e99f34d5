"""The operators around the retention core where they are used: rotary
positions inside MultiScaleRetention, the residual-norm seam as a module and in
a training step, the filtered draw inside the engine's generation, and all of
them in one small decoder.

Tolerances are the framework's own for its paths: fp32 1e-4, bf16 tensor-core
products 2e-2 of the largest value.
"""
import numpy as np
import pytest
import torch

from conftest import rel_err
from oracle import layer_ops_ref as L
from oracle import retention_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _module(d, H, seed, gated, **rot):
    import aceflow_b200 as af

    rng = np.random.default_rng(seed)
    m = af.nn.MultiScaleRetention(d, H, gated=gated, rotary=af.nn.Rotary(d // H, **rot))
    bf = lambda a: torch.from_numpy(a.astype(np.float32)).bfloat16().float().numpy()  # noqa: E731
    for n in ("w_q", "w_k", "w_v", "w_o") + (("w_g",) if gated else ()):
        setattr(m, n, af.nn.Parameter(af.Tensor(bf(0.03 * rng.standard_normal((d, d))))))
    return m


def _reference(m, x, position):
    """The layer in float64: rotation, retention in its parallel form, norm (or
    group norm and gate), output projection."""
    f = lambda p: p.numpy().astype(np.float64)  # noqa: E731
    B, T, d = x.shape
    H, D = m.num_heads, m.head_dim
    heads = lambda w: (x @ f(w).T).reshape(B, T, H, D)  # noqa: E731
    turn = lambda a: L.rotary64(a, m.rotary.inv_freq.numpy(), position, m.rotary.layout, m.rotary.scale)  # noqa: E731
    q, k, v = turn(heads(m.w_q)), turn(heads(m.w_k)), heads(m.w_v)
    dist = np.arange(T)[:, None] - np.arange(T)[None]
    decay = np.where(dist >= 0, m.gamma.astype(np.float64)[:, None, None] ** np.maximum(dist, 0), 0.0)
    o = np.einsum("bihd,bjhd,hij,bjhe->bihe", q, k, decay, v, optimize=True).reshape(B, T, d)
    if m.gated:
        n = R.group_norm_gate64(o.reshape(B * T, d), (x @ f(m.w_g).T).reshape(B * T, d), H,
                                f(m.group_norm_weight), f(m.group_norm_bias), m.ret_norm.eps).reshape(B, T, d)
    else:
        n = o / np.sqrt((o * o).mean(-1, keepdims=True) + m.ret_norm.eps)
    return n @ f(m.w_o).T


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rot", [dict(), dict(layout="half", rotary_dim=64, scaling="yarn", factor=4.0,
                                              original_length=2048)])
def test_retention_with_rotary_prompt_and_decode(dev, gated, rot):
    """Exact prefill, tensor-core prefill from a later position, and the state
    handed to decode steps, all against one float64 evaluation."""
    import aceflow_b200 as af

    B, T, d, H = 2, 90, 512, 2
    m = _module(d, H, 7, gated, **rot).to("cuda:0")
    x = torch.from_numpy(np.random.default_rng(8).standard_normal((B, T, d)).astype(np.float32)).bfloat16()
    at = 5000
    ref = _reference(m, x.double().numpy(), at + np.arange(T))
    exact = m(af.Tensor(x.float(), device="cuda:0"), at)
    assert rel_err(exact.numpy(), ref) < 1e-4
    for chunk in (64, 128):
        xb = af.Tensor(x.to(dev), device="cuda:0", dtype="bfloat16")
        out, st = m.forward_chunkwise(xb, chunk=chunk, position=at)
        assert out.dtype == "bfloat16" and rel_err(out.numpy(), ref) < 2e-2
    f32, _ = m.forward_chunkwise(af.Tensor(x.float(), device="cuda:0"), position=np.arange(at, at + T))
    assert f32.dtype == "float32" and rel_err(f32.numpy(), ref) < 2e-2
    # a prompt of T - 6 tokens, then single tokens (fp32 from a zero state, and from the prompt's)
    cut = T - 6
    _, st = m.forward_chunkwise(af.Tensor(x[:, :cut].to(dev), device="cuda:0", dtype="bfloat16"), position=at)
    outs = []
    for t in range(cut, T):
        pos = torch.full((B,), at + t, dtype=torch.int32, device=dev) if t % 2 else at + t
        o, st = m.forward_recurrent(af.Tensor(x[:, t].float(), device="cuda:0"), st, pos)
        outs.append(o.numpy())
    assert rel_err(np.stack(outs, 1), ref[:, cut:]) < 2e-2
    st, outs = m.init_state(B), []
    for t in range(20):
        o, st = m.forward_recurrent(af.Tensor(x[:, t].float(), device="cuda:0"), st, np.array([at + t, at + t]))
        outs.append(o.numpy())
    assert rel_err(np.stack(outs, 1), ref[:, :20]) < 1e-4


def test_residual_norm_module(dev):
    import aceflow_b200 as af

    d = 320
    rng = np.random.default_rng(11)
    x, h, g = (rng.standard_normal((3, 7, d)).astype(np.float32) for _ in range(3))
    m = af.nn.ResidualNorm(d, layer_scale=0.25, alpha=1.5)
    m.post_weight = af.nn.Parameter(af.Tensor(1 + 0.1 * rng.standard_normal(d)))
    host = m(af.Tensor(x), af.Tensor(h), af.Tensor(g))
    m.to("cuda:0")
    z, y = m(*(af.Tensor(a, device="cuda:0") for a in (x, h, g)))
    ref, _ = L.seam64(x, h, g, m.post_weight.numpy(), m.scale.numpy(), m.pre_weight.numpy(), 1.5, 1e-6)
    for a, b, name in ((z, host[0], "z"), (y, host[1], "y")):
        assert rel_err(a.numpy(), ref[name]) < 1e-5 and rel_err(b.numpy(), ref[name]) < 1e-5
    z, y = m(af.Tensor(x, device="cuda:0"), af.Tensor(h, device="cuda:0", dtype="bfloat16"))
    assert z.dtype == "float32" and y.dtype == "bfloat16"


def _engine(dev, V=300, d=128, H=2, batch=3, layers=2):
    from aceflow_b200.engine import AceEngine

    rng = np.random.default_rng(21)
    w = lambda *s: (0.2 * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    e = AceEngine(layers, d, H, w(V, d), batch=batch)
    for i in range(layers):
        e.load_layer_weights(i, w(3 * d, d), w(d, d), w(2 * 256, d), w(d, 256), np.ones(d), np.ones(d))
    return e


def test_engine_generation_with_settings_per_stream(dev):
    """Every generated token is the oracle's draw from the step's logits, with
    the stream's own settings and its last 60 ids penalised."""
    e = _engine(dev)
    prompts = np.random.default_rng(22).integers(0, 300, (3, 55))
    n = 12
    u = np.random.default_rng(23).random((3, n)).astype(np.float32)
    kw = dict(temperature=[0.0, 0.8, 1.2], top_k=[0, 40, 0], top_p=[1.0, 0.9, 0.98], min_p=[0.0, 0.02, 0.001],
              repetition_penalty=[1.3, 1.1, 1.0])
    toks, logits = e.generate_batch(prompts, n, return_logits=True, uniforms=u, **kw)
    compared = 0
    for b in range(3):
        seen = list(prompts[b])
        for s in range(n):
            want, _, margin = L.sample64(logits[b, s], u[b, s], kw["temperature"][b], kw["top_k"][b], kw["top_p"][b],
                                         kw["min_p"][b], kw["repetition_penalty"][b], seen[-60:])
            if margin > 1e-7:
                compared += 1
                assert toks[b, s] == want
            seen.append(int(toks[b, s]))
    assert compared > 30
    e.reset_memory()
    same = e.generate_batch(prompts, n, uniforms=u, **kw)
    assert np.array_equal(same, toks)
    with pytest.raises(ValueError, match="top_p"):
        e.generate_batch(prompts, 2, temperature=1.0, top_p=[0.5, 0.6])
    with pytest.raises(ValueError, match="positive"):
        e.generate_batch(prompts, 2, temperature=1.0, repetition_penalty=[1.0, 0.0, 1.0])
    lg = np.random.default_rng(24).standard_normal(300).astype(np.float32)
    assert e.sample_token_from_logits(lg, [], 1.0, 0, 1.0, 1.0, 0.7, min_p=0.3) == L.sample64(lg, 0.7, min_p=0.3)[0]
    big = np.random.default_rng(25).standard_normal(60000).astype(np.float32)  # more than af_sample_rows holds
    assert e.sample_token_from_logits(big, [], 1.0, 50, 0.9, 1.0, 0.7) == L.sample64(big, 0.7, 1.0, 50, 0.9)[0]


def test_a_decoder_of_all_of_them(dev):
    """Two layers (rotated retention, seam, SwiGLU, seam) over a prompt, then a
    token, logits and a draw: the prompt form in one go and token by token give
    the same residual stream, and the draw follows from the logits."""
    import aceflow_b200 as af
    from aceflow_b200 import cuda_ops

    B, T, d, H, V = 2, 33, 256, 2, 500
    np.random.seed(31)
    layers = [(af.nn.MultiScaleRetention(d, H, rotary=af.nn.Rotary(d // H)), af.nn.ResidualNorm(d, layer_scale=0.5),
               af.nn.SwiGLU(d, 512), af.nn.ResidualNorm(d, alpha=1.1)) for _ in range(2)]
    first, head = af.nn.RMSNorm(d), af.nn.Linear(d, V, bias=False)
    for m in (first, head, *(p for layer in layers for p in layer)):
        m.to("cuda:0")
    x = af.Tensor(np.random.randn(B, T, d).astype(np.float32), device="cuda:0")

    def run(x, retention):
        z, y = x, first(x)
        for i, (msr, seam1, ffn, seam2) in enumerate(layers):
            z, y = seam1(z, retention(i, msr, y))
            z, y = seam2(z, ffn(y))
        return z, y

    z, y = run(x, lambda i, msr, v: msr(v))
    states = [msr.init_state(B) for msr, *_ in layers]
    for t in range(T):
        def step(i, msr, v):
            out, states[i] = msr.forward_recurrent(v, states[i], t)
            return out

        zt, yt = run(af.Tensor(x.torch[:, t], device="cuda:0"), step)
        assert rel_err(zt.numpy(), z.numpy()[:, t]) < 1e-4
    logits = head(af.Tensor(y.torch[:, -1], device="cuda:0"))
    u = torch.tensor([0.2, 0.9], device=dev)
    tok = cuda_ops.sample_tokens(logits.torch, u, temperature=0.9, top_p=0.95, min_p=0.05).cpu().numpy()
    for b in range(B):
        want, _, margin = L.sample64(logits.numpy()[b], float(u[b]), 0.9, 0, 0.95, 0.05)
        assert margin < 1e-7 or tok[b] == want


def test_a_training_step_of_a_layer(dev):
    """Gradients of one layer (projection, rotation, chunkwise retention, W_o,
    gated seam) through the differentiable forms, bf16 activations, against
    float64 automatic differentiation of the plain formulas."""
    from aceflow_b200 import cuda_ops

    B, T, H = 2, 70, 2
    d = 256 * H
    g0 = torch.Generator(device=dev).manual_seed(41)
    r = lambda s, *shape: s * torch.randn(*shape, generator=g0, device=dev)  # noqa: E731
    bf = torch.bfloat16
    p = dict(x=r(1.0, B * T, d).to(bf), w_qkv=r(0.03, 3 * d, d).to(bf), w_o=r(0.03, d, d).to(bf),
             gate=r(1.0, B * T, d).to(bf), post=1 + r(0.1, d), scale=0.5 + r(0.05, d), pre=1 + r(0.1, d))
    cz, cy = r(1.0, B * T, d), r(1.0, B * T, d)
    gamma = cuda_ops.gammas(H, dev)
    freq, fs = cuda_ops.rotary_frequencies(256, device=dev)
    leaf = {k: v.clone().requires_grad_() for k, v in p.items()}
    qkv = leaf["x"] @ leaf["w_qkv"].t()
    qk = cuda_ops.rotary_autograd(qkv.view(B, T, 3 * H, 256)[:, :, :2 * H], freq, 11, scale=fs)
    turned = torch.cat([qk.reshape(B * T, 2 * d), qkv[:, 2 * d:]], 1)
    o = cuda_ops.retention_chunkwise_autograd(turned, B, T, H, gamma)
    z, y = cuda_ops.residual_norm_autograd(leaf["x"], o @ leaf["w_o"].t(), gate=leaf["gate"], post_w=leaf["post"],
                                           scale=leaf["scale"], pre_w=leaf["pre"])
    ((z * cz).sum() + (y * cy).sum()).backward()

    ref = {k: v.double().requires_grad_() for k, v in p.items()}
    q, k, v = (ref["x"] @ ref["w_qkv"].t()).view(B, T, 3, H, 256).unbind(2)
    th = (11 + torch.arange(T, device=dev, dtype=torch.float64))[:, None, None] * freq.double()

    def turn(a):
        e, f = a[..., 0::2], a[..., 1::2]
        return torch.stack((e * th.cos() - f * th.sin(), e * th.sin() + f * th.cos()), -1).flatten(-2)

    dist = torch.arange(T, device=dev)[:, None] - torch.arange(T, device=dev)[None]
    decay = torch.where(dist >= 0, gamma.double()[:, None, None] ** dist.clamp_min(0), 0.0)
    s = torch.einsum("bihd,bjhd->bhij", turn(q), turn(k)) * decay
    h = torch.einsum("bhij,bjhd->bihd", s, v).reshape(B * T, d) @ ref["w_o"].t()
    norm = lambda a, w: a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
    zr = ref["x"] + ref["scale"] * torch.nn.functional.silu(ref["gate"]) * norm(h, ref["post"])
    ((zr * cz.double()).sum() + (norm(zr, ref["pre"]) * cy.double()).sum()).backward()
    for name in p:
        assert rel_err(leaf[name].grad.double().cpu().numpy(), ref[name].grad.cpu().numpy()) < 2e-2, name


def test_a_captured_training_step(dev):
    """Forward and backward of rotation and seam captured into two graphs of
    different leaves and replayed in turn give the eager gradients."""
    from aceflow_b200 import cuda_ops

    freq, _ = cuda_ops.rotary_frequencies(64, device=dev)

    def leaves(rows, seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return [torch.randn(*s, generator=g, device=dev).requires_grad_()
                for s in ((rows, 320), (rows, 320), (rows, 320), (320,), (320,), (320,))]

    def grads(t):
        h = cuda_ops.rotary_autograd(t[1].view(-1, 5, 64), freq, 3).reshape(t[1].shape)
        z, y = cuda_ops.residual_norm_autograd(t[0], h, gate=t[2], post_w=t[3], scale=t[4], pre_w=t[5])
        return torch.autograd.grad((z * y).sum(), t)

    sets, graphs = [leaves(40, 1), leaves(700, 2)], []
    want = [[g.clone() for g in grads(t)] for t in sets]
    for t in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = grads(t)
        graphs.append((graph, out))
    for _ in range(2):
        for graph, _out in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        for a, b in zip(out, ref):
            assert torch.equal(a, b)


def test_rotary_frequencies_may_be_replaced(dev):
    import aceflow_b200 as af

    rot = af.nn.Rotary(64)
    x = af.Tensor(np.random.default_rng(3).standard_normal((2, 3, 64)).astype(np.float32), device="cuda:0")
    first = rot(x, 5).numpy()
    rot.inv_freq *= 0.5
    second = rot(x, 5).numpy()
    rot.inv_freq = rot.inv_freq * 2.0
    assert not np.array_equal(first, second) and np.array_equal(first, rot(x, 5).numpy())
