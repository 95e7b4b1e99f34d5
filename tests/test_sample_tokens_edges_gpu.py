"""Rows of the filtered draw (af_sample_tokens) where a cluster's exchanges, its
small weights and its settings go wrong first."""
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


@pytest.mark.parametrize("rows,V", [(3, 4100), (5, 8200), (9, 40000), (600, 20001), (500, 50000), (400, 131072)])
def test_every_block_hears_of_a_maximum_in_every_other(dev, rows, V):
    """2, 4 and 8 CTAs a row, a wave and many: the one large logit of a row moves
    through all slices; greedy and by mass."""
    from aceflow_b200 import cuda_ops

    at = (torch.arange(rows, device=dev) * 104729) % V
    lg = torch.full((rows, V), -60.0, device=dev)
    lg.scatter_(1, at[:, None], 3.0)
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(V), device=dev)
    for kw in (dict(temperature=0.0), dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.5)):
        tok, logp = cuda_ops.sample_tokens(lg, u, return_logprobs=True, **kw)
        assert torch.equal(tok.long(), at), kw
        assert torch.all(logp.abs() < 1e-6)  # what is left weighs V exp(-63) at most


# A mass is off by at most the larger of 2^-29 of itself and 2^-45 of the largest
# weight, so the mass of what is kept by 2^-29 + vocab 2^-45 of the row, and its
# logarithm by the same; the result is rounded to fp32.
def _mass_error(V):
    return 2.0 ** -29 + V * 2.0 ** -45


@pytest.mark.parametrize("kw", [dict(), dict(top_k=200), dict(top_p=0.9999999), dict(temperature=0.5)])
@pytest.mark.parametrize("V", [301, 4001, 131001])
def test_min_p_among_small_weights(dev, V, kw):
    """Half of a row's tokens 1e-5 above a min-p of 2^-30 and half as far below it:
    a weight of 2^-30 is a whole number of units of 2^-44 to 3e-5 of itself only."""
    from aceflow_b200 import cuda_ops

    temp, min_p = kw.get("temperature", 1.0), float(np.float32(2.0 ** -30))
    top = np.float32(temp * 20.794415)
    edge = float(top) + temp * np.log(min_p)
    row = np.full(V, edge + 1e-5 * temp, np.float32)
    row[1::2] = edge - 1e-5 * temp
    row[V // 2] = top
    want, logp, margin = L.sample64(row, 0.5, temp, kw.get("top_k", 0), kw.get("top_p", 1.0), min_p)
    above = int((row > edge).sum()) - 1
    kept = min(above, kw.get("top_k", V) - 1)
    if "top_p" not in kw:
        assert abs(logp + np.log1p(kept * np.exp(1e-5) * min_p)) < 1e-3 * kept * min_p
    tok, got = cuda_ops.sample_tokens(torch.from_numpy(row[None]).to(dev), torch.tensor([0.5], device=dev), min_p=min_p,
                                      return_logprobs=True, **kw)
    assert tok.item() == want == V // 2
    assert abs(got.item() - logp) <= _mass_error(V) + 2.0 ** -24 * abs(logp)


@pytest.mark.parametrize("min_p", [0.3, 1e-3, 1e-9, 3e-14])
def test_min_p_of_any_size(dev, min_p):
    """Weights spread over some octaves on either side of min-p; every row is
    compared unless its own border is nearer than its masses' error."""
    from aceflow_b200 import cuda_ops

    rng = np.random.default_rng(3)
    rows, V = 24, 20000
    lg = (np.log(min_p) + 1.5 * rng.standard_normal((rows, V))).astype(np.float32)
    lg[np.arange(rows), rng.integers(0, V, rows)] = 0.0
    lg = np.minimum(lg, 0.0)
    u = rng.random(rows).astype(np.float32)
    tok, got = cuda_ops.sample_tokens(torch.from_numpy(lg).to(dev), torch.from_numpy(u).to(dev), min_p=min_p,
                                      return_logprobs=True)
    compared = 0
    for r in range(rows):
        want, logp, _ = L.sample64(lg[r], u[r], min_p=min_p)
        w = np.exp(lg[r].astype(np.float64))
        share = np.sort(w[w >= float(np.float32(min_p))])[::-1].cumsum()
        if share.size > 1 and np.min(np.abs(share[:-1] / share[-1] - float(u[r]))) < _mass_error(V):
            continue
        compared += 1
        assert tok[r].item() == want
        assert abs(got[r].item() - logp) <= _mass_error(V) + 2.0 ** -23 * max(1.0, abs(logp))
    assert compared >= 12


@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.95), dict(min_p=0.02),
                                dict(temperature=0.7, top_k=40, top_p=0.9), dict(temperature=30.0),
                                dict(temperature=0.01), dict(top_k=20000, top_p=0.999, min_p=1e-6)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_row_under_each_filter(dev, kw, dtype):
    """Twenty draws of one row alone.  Both sides of a share are off by the masses'
    error at most, so a share by twice that (6e-9 here): a draw whose deciding
    border is nearer is left out, and so may be two in twenty at most."""
    from aceflow_b200 import cuda_ops

    rng = np.random.default_rng(len(str(kw)))
    lg = torch.from_numpy(3.0 * rng.standard_normal((1, 32000)).astype(np.float32)).to(dev).to(dtype)
    row = lg.float().cpu().numpy()[0]
    args = [kw.get(k, v) for k, v in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))]
    compared = 0
    for u in rng.random(20).astype(np.float32):
        tok, logp = cuda_ops.sample_tokens(lg, torch.tensor([u], device=dev), return_logprobs=True, **kw)
        want, ref, _ = L.sample64(row, u, *args)
        if _share_margin(row, u, *args) < 2 * _mass_error(32000):
            continue
        compared += 1
        assert tok.item() == want and abs(logp.item() - ref) <= 2e-7 * max(1.0, abs(ref))
    assert compared >= 18


def _share_margin(row, u, temperature, top_k, top_p, min_p):
    """How far, in shares of the mass that decides, u's draw and the crossing of
    top_p lie from the borders next to them (min-p is decided without sums)."""
    x = np.sort(row.astype(np.float64))[::-1]
    w = np.exp((x[:top_k] if top_k else x) - x[0]) if temperature == 1.0 else np.exp(
        ((x[:top_k] if top_k else x) - x[0]) / float(np.float32(temperature)))
    run, keep, margin = np.cumsum(w), w.size, 1.0
    if top_p < 1.0:
        p = float(np.float32(top_p))
        keep = 1 + int(np.searchsorted(run, p * run[-1], side="right"))
        margin = float(np.min(np.abs(run / run[-1] - p)))
    keep = min(keep, int((w >= float(np.float32(min_p))).sum()))
    return min(margin, float(np.min(np.abs(run[:keep - 1] / run[keep - 1] - float(u)), initial=1.0)))


def test_a_top_k_beyond_31_bits(dev):
    from aceflow_b200 import cuda_ops

    lg = 2.5 * torch.randn(30, 9000, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    u = torch.rand(30, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    want = cuda_ops.sample_tokens(lg, u)
    assert torch.equal(cuda_ops.sample_tokens(lg, u, top_k=2 ** 32 + 1), want)
    assert torch.equal(cuda_ops.sample_tokens(lg, u, top_k=-2 ** 32 + 1), want)
    assert not torch.equal(cuda_ops.sample_tokens(lg, u, top_k=1), want)
