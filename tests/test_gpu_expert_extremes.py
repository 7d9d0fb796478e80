"""fp32 products of finite values that bfloat16 alone would round to infinity (above 3.3895e38)."""
import pytest
import torch

from mace_onegpu import _native as N
from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu

BIG = [3.39e38, -3.4e38, 3.4028234e38]


@pytest.mark.parametrize("big", BIG)
def test_the_largest_fp32_values_are_values(big):
    """Products with factors of about 1e-3: results within fp32, with fp32 errors (the bound of the other products' tests)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T, E, D, O = 70, 2, 64, 48
    x = torch.randn(T, D, device="cuda", generator=g)
    w = torch.randn(E, O, D, device="cuda", generator=g) * 1e-3
    dy = torch.randn(T, 1, O, device="cuda", generator=g) * 1e-3
    x[7, 3] = big
    ex = torch.randint(0, E, (T, 1), device="cuda", generator=g, dtype=torch.int32)
    xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
    plan = X.plan_experts(ex, E)
    out = X.expert_linear(xd, wd, plan)
    dw, = torch.autograd.grad(out, wd, dy)
    few = N.ops().expert_linear(x, w, plan.experts, None, None)
    e = ex[:, 0].long()
    want = torch.einsum("td,tod->to", x.double(), w.double()[e])
    mag = torch.einsum("td,tod->to", x.double().abs(), w.double().abs()[e])
    for got in (out[:, 0].detach(), few[:, 0]):
        assert torch.isfinite(got).all()
        assert ((got.double() - want).abs() <= 16 * 2.0 ** -23 * mag).all()
    want, mag = torch.zeros(2, E, O, D, dtype=torch.float64, device="cuda")
    for i in range(E):
        t = torch.nonzero(e == i)[:, 0]
        want[i] = dy[t, 0].double().T @ x[t].double()
        mag[i] = dy[t, 0].double().abs().T @ x[t].double().abs()
    assert torch.isfinite(dw).all() and ((dw.double() - want).abs() <= 17 * 2.0 ** -23 * mag).all()
    # as a matrix, and as an upstream gradient
    w2 = torch.randn(E, O, D, device="cuda", generator=g)
    w2[1, 5, 9] = big
    x2 = torch.randn(T, D, device="cuda", generator=g) * 1e-3
    up = torch.randn(T, 1, O, device="cuda", generator=g) * 1e-3
    x2 = x2.requires_grad_()
    out = X.expert_linear(x2, w2, plan)
    dx, = torch.autograd.grad(out, x2, up)
    assert torch.isfinite(out).all() and torch.isfinite(dx).all()
    want = torch.einsum("to,tod->td", up[:, 0].double(), w2.double()[e])
    mag = torch.einsum("to,tod->td", up[:, 0].double().abs(), w2.double().abs()[e])
    assert ((dx.double() - want).abs() <= 16 * 2.0 ** -23 * mag).all()
