"""Layer norm of rows near the largest width (2^31 - 1 columns): the kernels' column counters step past it."""
import pytest
import torch

from mace_onegpu import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [2 ** 30 + 3, 2 ** 31 - 1])
def test_the_widest_rows(d):
    """Values +1 and -1 in turn: the mean is 1 / d, the variance 1 - 1 / d^2, and every result rounds to the value itself.
    dy = 1 in the first and last columns: dx = dy but for terms of 1 / d, db = dy, dw = dy xh."""
    x = torch.ones(1, d, dtype=torch.bfloat16, device="cuda")
    x[:, 1::2] = -1
    y, mean, rstd = N.ops().layer_norm_fwd(x, None, None, 1e-5)
    assert torch.equal(y, x)
    assert abs(float(mean)) <= 1e-6 and abs(float(rstd) - 1) <= 1e-5
    del y
    dy = torch.zeros_like(x)
    dy[0, :3] = 1
    dy[0, -3:] = 1
    dx, dw, db = N.ops().layer_norm_bwd(dy, x, None, mean, rstd, True, True, True, False)
    assert torch.equal(db, dy[0]) and torch.equal(dw, (dy * x)[0])
    # the means of dy and of dy xh are below 6 / d = 6e-9
    assert torch.equal(dx[0, :3], dy[0, :3]) and torch.equal(dx[0, -3:], dy[0, -3:])
    assert float(dx[0, 3:-3].abs().max()) <= 2e-8
