"""Rows of any alignment that stay in registers, at both ends of every number of pieces of 128 values and just beyond the last."""
import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
WIDTHS = sorted({w + d for w in range(0, 1152, 128) for d in (-1, 0, 1) if w + d > 0})


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", WIDTHS)
def test_widths(k, dt):
    g = torch.Generator(device="cuda").manual_seed(k)
    x = (torch.randn(37, k + 4, generator=g, device="cuda") * 3).to(dt)[:, 1:k + 1]   # rows that start off any vector
    q, s = X.quantize_rows(x)
    top = x.float().abs().amax(1).cpu()                       # (on the GPU torch divides by a number as a product)
    assert torch.equal(s.cpu(), top / 127) and q.stride(0) % 16 == 0
    assert torch.equal(q.double(), torch.round(x.double() / s.double()[:, None]))      # nearest, ties to even
    full = q.as_strided((37, q.stride(0)), (q.stride(0), 1))
    assert not full[:, k:].any()
