"""GPU test of hc_read_norm where a token holds an infinity: the mean square is
infinite, its inverse root 0, so that RMS gives the bias in every finite place
and NaN in the infinite ones, for each number of blocks and on every path."""

import pytest
import torch

from tests.test_block_gpu import ops, read_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 4, 8])
@pytest.mark.parametrize("m", [1, 2, 3, 4])
@pytest.mark.parametrize("D", [64, 333, 512])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_rms_of_an_infinite_token(n, m, D, dt):
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    R, x, w, b, _ = read_inputs(5, n, m, D, dt, "wb")
    want = ops().hc_read_norm(R, x, w, b)
    x[2, 1, 7] = float("inf")
    y = ops().hc_read_norm(R, x, w, b)
    assert torch.equal(y[[0, 1, 3, 4]], want[[0, 1, 3, 4]])
    place = torch.zeros(m, D, dtype=torch.bool, device="cuda")
    place[:, 7] = True
    assert y[2][place].isnan().all()
    assert torch.equal(y[2][~place], b.view(m, D)[~place].to(x.dtype))
