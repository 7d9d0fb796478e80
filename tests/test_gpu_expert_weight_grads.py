"""Gradients of the experts' matrices from 16-bit data with routing weights: the weights are fp32 numbers of any size, and
weight times row keeps enough bits that the result is rounded once; long sums over one expert do not shrink."""
import pytest
import torch

from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu


def _exact_dw(x, ex, p, dy, E):
    """dW [E, O, D] in 64 bits; x [T, D] or [T, k, D], p [T, k]."""
    T, k = ex.shape
    x, dy, p = x.double(), dy.double(), p.double()
    dw = torch.zeros(E, dy.shape[-1], x.shape[-1], dtype=torch.float64, device=x.device)
    for e in range(E):
        for j in range(k):
            t = torch.nonzero(ex[:, j] == e)[:, 0]
            dw[e] += (p[t, j, None] * dy[t]).T @ (x[t, j] if x.dim() == 3 else x[t])
    return dw


def _grad(x, w, ex, p, dy):
    w = w.requires_grad_()
    plan = X.plan_experts(ex, w.shape[0])
    dw, = torch.autograd.grad(X.expert_linear(x, w, plan, p), w, dy)
    plan.check()
    return dw


def _one_rounding(got, exact, slack=1.05):
    exact = exact.cpu()
    mine = (got.double().cpu() - exact).norm()
    best = (exact.to(got.dtype).double() - exact).norm()
    assert mine <= slack * best, float(mine / best)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,E,D,O,slots", [(900, 2, 5, 192, 136, False), (2500, 4, 6, 256, 264, False), (700, 3, 4, 72, 515, True),
                                             (901, 1, 9, 130, 77, False), (30, 2, 40, 64, 64, False)])
def test_weighted_gradient_is_rounded_once(T, k, E, D, O, slots, dt):
    """Weight times row is carried to 2^-16 of itself, so that the final rounding to the type is the error that counts."""
    g = torch.Generator(device="cuda").manual_seed(T + k)
    x = torch.randn(*((T, k, D) if slots else (T, D)), device="cuda", generator=g).to(dt)
    w = torch.zeros(E, O, D, device="cuda", dtype=dt)
    ex = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    ex[::7, 0] = -1
    p = torch.rand(T, k, device="cuda", generator=g) + 0.1
    dy = torch.randn(T, O, device="cuda", generator=g).to(dt)
    _one_rounding(_grad(x, w, ex, p, dy), _exact_dw(x, ex, p, dy, E))


@pytest.mark.parametrize("weight,xs,dys", [(1e-4, 1.0, 1.0), (1e-7, 1.0, 1e4), (1e-9, 1e3, 1e4), (1e3, 100.0, 1e-3), (1e5, 10.0, 1e-4),
                                           (1e10, 1e-4, 1e-7)])
def test_weighted_gradient_over_the_range_of_the_weights(weight, xs, dys):
    """fp16: weight times row may lie far outside the type's range where the gradient does not."""
    g = torch.Generator(device="cuda").manual_seed(7)
    T, k, E, D, O = 300, 2, 3, 64, 72
    x = (torch.randn(T, D, device="cuda", generator=g) * xs).half()
    dy = (torch.randn(T, O, device="cuda", generator=g) * dys).half()
    assert torch.isfinite(x).all() and torch.isfinite(dy).all()
    ex = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    p = (torch.rand(T, k, device="cuda", generator=g) + 0.5) * weight
    want = _exact_dw(x, ex, p, dy, E)
    assert want.abs().max() < 6e4
    dw = _grad(x, torch.zeros(E, O, D, device="cuda", dtype=torch.float16), ex, p, dy)
    assert torch.isfinite(dw).all()
    _one_rounding(dw, want)
