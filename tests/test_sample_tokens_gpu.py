"""The filtered draw (af_sample_tokens) against a float64 evaluation.

The kernel's masses are whole numbers of 2^-44 of the largest weight, each off
by less than 2^-29 of itself: a row whose deciding border lies within 1e-7 of
its draw (the oracle reports the distance) is not compared, every other one
gives the same token.  The log-probability is an fp32 rounding of a value off
by less than 1e-7.
"""
import numpy as np
import pytest
import torch

from oracle import layer_ops_ref as L

pytestmark = pytest.mark.gpu

MARGIN = 1e-7


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _draw(dev, logits, u, dtype=torch.float32, **kw):
    from aceflow_b200 import cuda_ops

    lt = torch.as_tensor(np.asarray(logits, np.float32)).to(dev).to(dtype)
    ut = torch.as_tensor(np.asarray(u, np.float32)).to(dev)
    for k, v in list(kw.items()):
        if isinstance(v, (list, np.ndarray)):
            dt = torch.int32 if k in ("top_k", "context") else torch.float32
            kw[k] = torch.as_tensor(np.asarray(v)).to(dev, dt)
    tok, lp = cuda_ops.sample_tokens(lt, ut, return_logprobs=True, **kw)
    return tok.cpu().numpy(), lp.cpu().numpy(), lt.float().cpu().numpy()


def _check(dev, logits, u, dtype=torch.float32, need=0.9, **kw):
    tok, lp, lg = _draw(dev, logits, u, dtype, **dict(kw))
    at = lambda v, r: v[r] if isinstance(v, (list, np.ndarray)) else v  # noqa: E731
    compared = 0
    for r in range(len(tok)):
        want, logp, margin = L.sample64(lg[r], u[r], at(kw.get("temperature", 1.0), r), at(kw.get("top_k", 0), r),
                                        at(kw.get("top_p", 1.0), r), at(kw.get("min_p", 0.0), r),
                                        at(kw.get("repetition_penalty", 1.0), r),
                                        kw["context"][r] if kw.get("context") is not None else ())
        if margin < MARGIN:
            continue
        compared += 1
        assert tok[r] == want, (r, tok[r], want, margin)
        assert lp[r] == logp or abs(lp[r] - logp) <= 2e-7 * max(1.0, abs(logp)), (r, lp[r], logp)
    assert compared >= need * len(tok)


def test_hand_worked_draws(dev):
    """Probabilities .1 .2 .3 .4."""
    lg = np.log(np.array([1.0, 2.0, 3.0, 4.0], np.float32))
    t4 = lambda us, **kw: _draw(dev, np.tile(lg, (len(us), 1)), us, **kw)[0].tolist()  # noqa: E731
    assert t4([0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91]) == [3, 3, 2, 2, 1, 1, 0]
    assert t4([0.56, 0.58], top_k=2) == [3, 2]
    assert t4([0.99], top_p=0.5) == [2] and t4([0.99], top_p=0.3) == [3]
    assert t4([0.99], min_p=0.6) == [2] and t4([0.99], min_p=0.45) == [1] and t4([0.99], min_p=1.0) == [3]
    assert t4([0.5, 0.99], temperature=0.0) == [3, 3]
    assert t4([0.5, 0.7], repetition_penalty=2.0, context=[[3, 3], [3, 3]]) == [1, 3]
    lp = _draw(dev, [lg], [0.99], min_p=0.6)[1]
    assert abs(lp[0] - np.log(3 / 7)) < 2e-7


@pytest.mark.parametrize("V", [1, 2, 31, 33, 500, 2047, 32000, 50257, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabularies_with_settings_per_row(dev, V, dtype):
    rng = np.random.default_rng(V)
    rows = 24 if V < 100000 else 10
    logits = 2.5 * rng.standard_normal((rows, V))
    pick = lambda v: np.asarray(v)[rng.integers(0, len(v), rows)]  # noqa: E731
    # a bf16 row has many equal logits and few distinct borders: a draw may fall nearer to one
    _check(dev, logits, rng.random(rows), dtype, need=0.8, temperature=pick([0.0, 0.3, 0.8, 1.0, 1.7]),
           top_k=pick([0, 0, 1, 7, 40, 1000, V, V + 5]), top_p=pick([1.0, 0.99, 0.9, 0.5, 0.0]),
           min_p=pick([0.0, 0.0, 0.001, 0.05, 0.7, 1.0]))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.95), dict(min_p=0.02),
                                dict(temperature=0.7, top_k=40, top_p=0.9), dict(temperature=30.0),
                                dict(temperature=0.01), dict(top_k=20000, top_p=0.999, min_p=1e-6)])
@pytest.mark.parametrize("rows,V", [(1, 32000), (70, 4001)])
def test_each_filter(dev, kw, rows, V):
    rng = np.random.default_rng(rows + V)
    _check(dev, 3.0 * rng.standard_normal((rows, V)), rng.random(rows), need=0.8 if rows > 1 else 0.0, **kw)


def test_equal_logits_lowest_index_first(dev):
    us = np.array([0.05, 0.25, 0.45, 0.65, 0.85])
    z = np.zeros((5, 9000))
    assert _draw(dev, z, us, top_k=5)[0].tolist() == [0, 1, 2, 3, 4]
    assert _draw(dev, z, us)[0].tolist() == [int(np.ceil(u * 9000 - 1e-6)) - 1 for u in np.float32(us).astype(float)]
    assert _draw(dev, z, us, temperature=0.0)[0].tolist() == [0] * 5
    two = np.full((2, 300), -1.0)
    two[:, 7] = two[:, 200] = 4.0
    assert _draw(dev, two, [0.4, 0.6], min_p=0.9)[0].tolist() == [7, 200]
    signed = np.array([[-0.0, 0.0, -1.0], [0.0, -0.0, -1.0]])  # the zeros are equal
    assert _draw(dev, signed, [0.2, 0.2], top_k=2)[0].tolist() == [0, 0]
    assert _draw(dev, signed, [0.7, 0.7], top_k=2)[0].tolist() == [1, 1]


def test_masked_rows_infinities_and_nan(dev):
    inf, nan, low = np.inf, np.nan, np.finfo(np.float32).min
    lg = np.array([[-inf] * 6, [nan, -inf, nan, -inf, -inf, nan], [-inf, 1.0, -inf, nan, 1.0, -inf],
                   [inf, 1.0, inf, 2.0, -inf, nan], [low] * 6, [low, 3.0, low, low, -inf, low],
                   [-inf, -inf, -inf, -inf, -inf, -5.0]])
    u = [0.6] * 7
    for kw in (dict(), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=4), dict(temperature=0.0)):
        tok, lp, _ = _draw(dev, lg, u, **kw)
        greedy = kw.get("temperature") == 0.0
        assert tok[0] == tok[1] == -1 and np.isneginf(lp[:2]).all()
        assert tok[2] == (1 if greedy else 4) and tok[3] == (0 if greedy else 2)
        assert tok[4] == (0 if greedy else {4: 2}.get(kw.get("top_k"), 3)) and tok[5] == 1 and tok[6] == 5
        if not greedy:
            assert abs(lp[2] - np.log(0.5)) < 1e-6 and abs(lp[3] - np.log(0.5)) < 1e-6 and abs(lp[5]) < 1e-6


def test_context_penalty(dev):
    """Repeated, padded and out-of-range ids; a penalty per row; rows without."""
    rng = np.random.default_rng(5)
    rows, V = 16, 5003
    logits = (3.0 * rng.standard_normal((rows, V))).astype(np.float32)
    ctx = rng.integers(0, V, (rows, 300)).astype(np.int32)
    ctx[:, :40] = ctx[:, 40:80]
    ctx[:, -7:] = -1
    ctx[0, 0], ctx[1, 1] = V, 2 ** 31 - 1
    for r in range(rows):
        logits[r, ctx[r, 100]] = 20.0
    pen = np.where(np.arange(rows) % 3 == 0, 1.0, 1.0 + rng.random(rows)).astype(np.float32)
    _check(dev, logits, rng.random(rows), repetition_penalty=pen, context=ctx, top_p=0.95, temperature=1.1)
    _check(dev, logits, rng.random(rows), repetition_penalty=1.3, context=ctx, temperature=0.0)


def test_borders_of_the_uniform_number(dev):
    lg = np.log(np.array([[1.0, 2.0, 3.0, 4.0]] * 4, np.float32))
    assert _draw(dev, lg, [0.0, 1.0, -3.0, np.float32(1 - 2.0 ** -24)])[0].tolist() == [3, 0, 3, 0]


def test_row_strides_batch_independence_streams_and_graphs(dev):
    from aceflow_b200 import cuda_ops

    V = 7001
    wide = torch.randn(40, V + 13, device=dev) * 3
    lg, u = wide[:, 5:5 + V], torch.rand(40, device=dev)
    kw = dict(top_p=0.97, min_p=0.001)
    want = cuda_ops.sample_tokens(lg.contiguous(), u, **kw)
    assert torch.equal(cuda_ops.sample_tokens(lg, u, **kw), want)
    for r in (0, 17, 39):  # alone or in a batch: the same token
        assert torch.equal(cuda_ops.sample_tokens(lg[r:r + 1], u[r:r + 1], **kw), want[r:r + 1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = cuda_ops.sample_tokens(lg, u, **kw)
    s.synchronize()
    assert torch.equal(again, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cuda_ops.sample_tokens(lg, u, **kw)
    u2 = torch.rand(40, device=dev)
    for v in (u2, u.clone()):
        u.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cuda_ops.sample_tokens(lg, v, **kw))
    assert cuda_ops.sample_tokens(lg[:0], u[:0]).numel() == 0


def test_agrees_with_the_one_setting_sampler(dev):
    """Where min_p is off, the same tokens as af_sample_rows (whose fp32 sums
    may pick a neighbour within 1e-4 of a border)."""
    from aceflow_b200 import cuda_ops

    lg = 3 * torch.randn(64, 32000, device=dev)
    u = torch.rand(64, device=dev)
    a = cuda_ops.sample_tokens(lg, u, temperature=0.8, top_k=60, top_p=0.95)
    b = cuda_ops.sample_rows(lg, u, temperature=0.8, top_k=60, top_p=0.95, repetition_penalty=1.0)
    for r in torch.nonzero(a != b).flatten().tolist():
        _, _, margin = L.sample64(lg[r].cpu().numpy(), float(u[r]), 0.8, 60, 0.95)
        assert margin < 1e-4


def test_places_in_crowded_bins(dev):
    """Bins of a sixteenth of an octave (0.043 of a logit at temperature 1) with
    more tokens than one CTA takes over at once (2048): two bins that are too
    many together, a crossing of top-p in a small bin before a draw in an
    overfull one, and the other way round."""
    rng = np.random.default_rng(77)
    wide = 2.5 * rng.standard_normal((4, 327680))
    # where top-p 0.95 is crossed a token weighs exp(2.1) / (327680 exp(3.1)) = 1.1e-6 of the row: 1e-7 on either
    # side leave 0.82 of the crossings and of the draws next to them, 0.67 of the rows
    _check(dev, wide, [0.97, 0.99, 0.9995, 0.5], need=0.5, top_p=[0.95, 0.97, 0.95, 1.0], min_p=[0.0, 0.0, 1e-6, 1e-5])
    head = 0.03 * rng.random((6, 3000))
    tail = -3.0 + rng.standard_normal((6, 20000))
    crowd = rng.permuted(np.concatenate([head, tail], 1), axis=1)
    _check(dev, crowd, [0.3, 0.6, 0.9, 0.97, 0.999, 0.2], need=0.6, top_p=[0.95, 0.9, 0.5, 0.97, 1.0, 0.3])
    _check(dev, crowd, [0.3, 0.6, 0.9, 0.97, 0.999, 0.2], need=0.6, min_p=[0.0, 0.97, 0.99, 0.02, 0.01, 0.5], top_p=0.99)


@pytest.mark.parametrize("rows,V", [(200, 5000), (160, 20001), (160, 50000)])
def test_many_rows_take_fewer_blocks_each(dev, rows, V):
    """The number of CTAs that share a row depends on both sizes (here one, two
    and four); the token does not."""
    rng = np.random.default_rng(V)
    pick = lambda v: np.asarray(v)[rng.integers(0, len(v), rows)]  # noqa: E731
    logits, u = 3.0 * rng.standard_normal((rows, V)), rng.random(rows)
    kw = dict(temperature=pick([0.0, 0.7, 1.2]), top_k=pick([0, 0, 30]), top_p=pick([1.0, 0.95, 0.6]),
              min_p=pick([0.0, 0.0, 0.02]))
    _check(dev, logits[:48], u[:48], **{k: v[:48] for k, v in kw.items()})
    many, few = _draw(dev, logits, u, **dict(kw)), _draw(dev, logits[:2], u[:2], **{k: v[:2] for k, v in kw.items()})
    assert (many[0][:2] == few[0]).all() and (many[1][:2] == few[1]).all()
    part = _draw(dev, logits[:48], u[:48], **{k: v[:48] for k, v in kw.items()})
    assert (many[0][:48] == part[0]).all() and (many[1][:48] == part[1]).all()


def test_offsets_beyond_31_bits(dev):
    """Logits with more than 2^31 values: the last rows draw as they do alone."""
    from aceflow_b200 import cuda_ops

    rows, V, last = 16400, 131072, 4
    g = torch.Generator(device=dev).manual_seed(9)
    lg = torch.zeros(rows, V, device=dev, dtype=torch.bfloat16)
    lg[-last:] = (2.5 * torch.randn(last, V, generator=g, device=dev)).bfloat16()
    u = torch.rand(rows, generator=g, device=dev)
    kw = dict(top_k=50, top_p=0.9, return_logprobs=True)
    many, few = cuda_ops.sample_tokens(lg, u, **kw), cuda_ops.sample_tokens(lg[-last:].clone(), u[-last:].clone(), **kw)
    assert torch.equal(many[0][-last:], few[0]) and torch.equal(many[1][-last:], few[1])
