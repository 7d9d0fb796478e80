"""8-bit products of tokens and weights at both ends of the range of the types: finite results are finite.

Tolerances.  Sums are exact, so y differs from (sum s_n) s_t + b in fp64 by two products' and one sum's roundings, 3 x 2^-24 of the
product, by the rounding to the type, and where the product is below the least normal number by half of the smallest subnormal."""
import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
CASES = [(torch.float32, 1e37, 1.0), (torch.bfloat16, 1e37, 1.0), (torch.float32, 1e-36, 1.0), (torch.bfloat16, 1e-36, 1.0),
         (torch.float16, 2e4, 0.5), (torch.float16, 1e-5, 1.0), (torch.float32, 1.0, 1e33), (torch.float32, 1.0, 1e-36),
         (torch.float32, 1e34, 1e-34), (torch.bfloat16, 1e-33, 1e33), (torch.float32, 1e30, 1e7), (torch.float32, 1e-20, 1e-17)]


@pytest.mark.parametrize("t", [1, 2, 4, 40, 700])
@pytest.mark.parametrize("dt,xs,ws", CASES)
def test_ends_of_the_range(t, dt, xs, ws):
    k, n = 272, 300
    g = torch.Generator(device="cuda").manual_seed(t)
    x = ((torch.rand(t, k, generator=g, device="cuda") * 2 - 1) * xs).to(dt)
    w = (torch.rand(n, k, generator=g, device="cuda") * 2 - 1) * (0.1 * ws)
    b = ((torch.rand(n, generator=g, device="cuda") - 0.5) * (xs * ws if xs * ws < 1e3 else 1.0)).to(dt)
    wq, wscale = X.quantize_rows(w)
    q, s = X.quantize_rows(x)
    sums = q.cpu().double() @ wq.cpu().double().T             # whole numbers below 2^53
    prod = sums * wscale.cpu().double() * s.cpu().double()[:, None]
    want = prod + b.cpu().double()
    assert want.abs().max() < torch.finfo(dt).max
    for y in (X.int8_linear(x, wq, wscale, b), X.int8_linear(q, wq, wscale, b, xscale=s, out_dtype=dt)):
        off = (y.cpu().double() - want).abs()
        tol = U[dt] * want.abs() + 4 * 2.0 ** -24 * (prod.abs() + want.abs()) * (1 + U[dt]) + LEAST[dt] + 2.0 ** -149 * s.cpu().double()[:, None]
        assert bool((off <= tol).all())
