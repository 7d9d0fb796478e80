"""Statistics of samples without rows: mean 0 and 1 / sqrt(eps), with and without rows elsewhere."""
import pytest
import torch

from mace_onegpu import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [1e-5, 0.25, 0.0])
@pytest.mark.parametrize("shape,off", [((0, 5, 16), None), ((4, 0, 16), None), ((0, 16), [0]), ((0, 16), [0, 0, 0]), ((6, 16), [2, 2]),
                                       ((6, 16), [6, 6, 6])])
def test_statistics_of_empty_samples(shape, off, eps):
    torch.full((4096,), float("nan"), device="cuda")           # (what freed memory may hold)
    x = torch.randn(*shape, device="cuda")
    y, mean, rstd = N.ops().group_norm_fwd(x, 4, None, None, eps, 1, None if off is None else torch.tensor(off).cuda())
    n = shape[0] if off is None else len(off) - 1
    assert mean.shape == rstd.shape == (n, 4) and not y.any() and not mean.any()
    # rsqrtf is 2 ulps off at most
    want = torch.full((n, 4), eps, device="cuda", dtype=torch.float32).double().rsqrt()
    assert bool(((rstd.double() == want) | ((rstd.double() - want).abs() <= 4 * 2.0 ** -24 * want)).all())
