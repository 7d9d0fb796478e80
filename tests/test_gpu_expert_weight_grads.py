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


def _skewed(T, E, D, O, dt, weighted, seed=3):
    """T slots, all but E of them on expert 0, with products of one sign; columns of different size, so that the sums spread
    over the steps of the type."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cx, cy = (torch.rand(n, device="cuda", generator=g) + 0.5 for n in (D, O))
    x = ((torch.rand(T, D, device="cuda", generator=g) + 0.5) * cx / 64).to(dt)
    dy = ((torch.rand(T, 1, O, device="cuda", generator=g) + 0.5) * cy).to(dt)
    ex = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    ex[:E, 0] = torch.arange(E, device="cuda")
    p = torch.rand(T, 1, device="cuda", generator=g) + 0.5 if weighted else None
    return x, dy[:, 0] if weighted else dy, ex, p


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("E", [1, 8, 640])
def test_long_sums_over_one_expert_do_not_shrink(E, weighted, dt):
    """400,000 rows on one expert, whatever the number of experts.  The tensor cores cut off what they add to an accumulator:
    sums of one sign lose 1e-7 for each 16 terms (measured: 2.5e-3 of this one when it is left alone).  5.3e-5 are 530 such steps.
    Rounding to the type has a deviation of u / sqrt(3) at most, u = 2^-8 or 2^-11: 4 u / sqrt(3 D O) is four deviations
    of the mean."""
    T, D, O = 400_000, 64, 72
    x, dy, ex, p = _skewed(T, E, D, O, dt, weighted)
    dw = _grad(x, torch.zeros(E, O, D, device="cuda", dtype=dt), ex, p, dy)
    z = dy.reshape(T, O).double() * (1.0 if p is None else p.double())
    on = ex[:, 0] == 0
    want = z[on].T @ x[on].double()
    assert want.abs().max() < 6e4
    mean = float(((dw[0].double() - want) / want).mean())
    u = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -11
    assert abs(mean) <= 5.3e-5 + 4 * u / (3 * D * O) ** 0.5, mean
    last = min(E - 1, 5)
    t = torch.nonzero(ex[:, 0] == last)[:, 0]
    want = z[t].T @ x[t].double()
    assert (dw[last].double() - want).norm() <= u * want.norm()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_very_wide_rows_do_not_shrink(dt):
    """The same for the products along the widths: 300,000 columns of one sign, forward (D) and dx (O)."""
    g = torch.Generator(device="cuda").manual_seed(5)
    wide, n, T = 300_000, 72, 50
    u = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -11
    a = ((torch.rand(T, wide, device="cuda", generator=g) + 0.5) * (torch.rand(T, 1, device="cuda", generator=g) + 0.5)).to(dt)
    c = ((torch.rand(1, n, wide, device="cuda", generator=g) + 0.5) * (torch.rand(1, n, 1, device="cuda", generator=g) + 0.5) / 64).to(dt)
    want = a.double() @ c[0].double().T
    plan = X.plan_experts(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), 1)
    fwd = X.expert_linear(a.requires_grad_(), c, plan)[:, 0].detach()
    x = torch.zeros(T, n, device="cuda", dtype=dt).requires_grad_()
    w = c.transpose(1, 2).contiguous()
    dx, = torch.autograd.grad(X.expert_linear(x, w, plan), x, a.detach()[:, None])
    plan.check()
    for got in (fwd, dx):
        mean = float(((got.double() - want) / want).mean())
        assert abs(mean) <= 5.3e-5 + 4 * u / (3 * T * n) ** 0.5, mean


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_infinities_in_a_weighted_gradient(dt):
    """An infinite x or dy gives what its products add up to: infinities of their sign, NaN where they meet zero or each other;
    the rest is untouched."""
    g = torch.Generator(device="cuda").manual_seed(9)
    T, k, E, D, O = 200, 2, 3, 64, 72
    x = torch.randn(T, D, device="cuda", generator=g).to(dt)
    dy = torch.randn(T, O, device="cuda", generator=g).to(dt)
    x[3, 5], x[9, 6], dy[20, 7], dy[3, 11] = float("inf"), -float("inf"), -float("inf"), 0.0
    ex = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    p = torch.rand(T, k, device="cuda", generator=g) + 0.1
    got = _grad(x, torch.zeros(E, O, D, device="cuda", dtype=dt), ex, p, dy)
    want = _exact_dw(x, ex, p, dy, E)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)].double(), want[torch.isinf(want)]) and torch.isinf(want).any()
    fine = torch.isfinite(want)
    assert fine.double().mean() > 0.9
    _one_rounding(got[fine], want[fine])
