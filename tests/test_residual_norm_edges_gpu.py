"""The residual-norm seam (af_residual_norm and its backward) at gates far from
zero and in views, where its precision and its strides go wrong first."""
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


@pytest.mark.parametrize("d", [40, 1000, 1531, 4100, 8192, 9001])
@pytest.mark.parametrize("ht", [F32, BF16])
def test_gates_far_from_zero_in_fp32(dev, d, ht):
    """z = swish(gate) where x is 0 and h 1.  CUDA's expf is off by at most 2 units
    (2 * 2^-23), the sum, the division and the product by half a one each (2^-24): below
    2^-22 + 3 * 2^-24 of the value."""
    from aceflow_b200 import cuda_ops

    g = torch.linspace(-80.0, 20.0, 7 * d, device=dev).view(7, d).to(ht)
    x, h = torch.zeros(7, d, device=dev), torch.ones(7, d, device=dev, dtype=ht)
    z, _ = cuda_ops.residual_norm(x, h, gate=g)
    ref = L.swish64(g.double().cpu().numpy())
    assert np.all(np.abs(z.double().cpu().numpy() - ref) <= (2.0 ** -22 + 3 * 2.0 ** -24) * np.abs(ref) * 1.01)
