"""gelu of group norm far from zero, relative to the value itself: with weights of zero z is the bias.

Tolerances.  One rounding to the type (half a step: 2^-24, 2^-8, 2^-11 of the value, and half of float16's smallest, 2^-25).  16-bit types
take the normal tail Phi(-|z|) from a polynomial that is 3e-6 off up to |z| = 5.5 and 4e-5 up to 13, times a power whose exponent
0.72 z^2 is rounded (2^-23 of it, 1e-5 at 13): 6e-5 of the tail.  float32 calls normcdff (CUDA gives 5 ulps) and expf on -z^2 / 2 rounded
twice (2^-23 of it).  The slope Phi(z) + z phi(z) has both terms' errors."""
import math

import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_tail(dt, sign):
    z = (sign * torch.linspace(0, 13, 8192, dtype=torch.float64)).float()
    b = z.cuda().requires_grad_()
    x = torch.randn(1, 1, 8192, device="cuda").to(dt)
    y = X.group_norm(x, 1, torch.zeros(8192, device="cuda"), b, activation="gelu")
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    z = z.double()
    cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    rel = 6e-5 if dt != torch.float32 else 8 * 2.0 ** -23
    rel = rel + 2.0 ** -23 * z * z                             # of the exponent
    want, slope = z * cdf, cdf + z * pdf
    off = (y.detach().cpu().double()[0, 0] - want).abs()
    tol = (U[dt] * (1 + rel) + rel) * want.abs() + LEAST[dt]
    assert bool((off <= tol).all()), float((off / want.abs())[off > tol].max())
    off = (db.cpu().double() - slope).abs()
    assert db.dtype == torch.float32
    assert bool((off <= (rel + 4 * 2.0 ** -24) * (cdf + z.abs() * pdf) + 2.0 ** -126).all())
