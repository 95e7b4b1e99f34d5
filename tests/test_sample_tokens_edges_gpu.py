"""Rows of the filtered draw (af_sample_tokens) where a cluster's exchanges, its
small weights and its settings go wrong first."""
import numpy as np
import pytest
import torch

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
