"""Expert products of 16-bit data whose rows are summed over k choices (the output, and dx): the sums are fp32 and rounded
once, so their error against 64 bits is that of rounding the exact result, and no single row has to fit the type."""
import pytest
import torch

from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu


def _exact(x, w, ex, p, dy):
    """out and dx in 64 bits on the GPU; p None: no weights (dy [T, k, O])."""
    T, k = ex.shape
    E, O, D = w.shape
    x, w, dy = x.double(), w.double(), dy.double()
    out = torch.zeros(T, O, dtype=torch.float64, device=x.device)
    dx = torch.zeros(T, D, dtype=torch.float64, device=x.device)
    for e in range(E):
        for j in range(k):
            t = torch.nonzero(ex[:, j] == e)[:, 0]
            g = torch.ones(len(t), 1, dtype=torch.float64, device=x.device) if p is None else p[t, j, None].double()
            out.index_add_(0, t, g * (x[t] @ w[e].T))
            dx.index_add_(0, t, g * ((dy[t] if p is not None else dy[t, j]) @ w[e]))
    return out, dx


def _one_rounding(got, exact, slack=1.05):
    """The 2-norm of the error is at most `slack` times that of rounding the exact value.  The fp32 arithmetic before it is
    (8 + K / 8) 2^-23 or better, below a twentieth of the rounding of fp16 for the K here, and adds in quadrature."""
    exact = exact.cpu()
    mine = (got.detach().double().cpu() - exact).norm()
    best = (exact.to(got.dtype).double() - exact).norm()
    assert mine <= slack * best, float(mine / best)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,E,D,O", [(700, 2, 5, 192, 136), (1500, 4, 6, 256, 264), (333, 3, 4, 72, 515), (901, 8, 9, 130, 77),
                                         (20_000, 2, 6, 192, 600)])
@pytest.mark.parametrize("weighted", [False, True])
def test_sums_over_choices_are_rounded_once(T, k, E, D, O, dt, weighted):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, D, device="cuda", generator=g).to(dt).requires_grad_()
    w = (torch.randn(E, O, D, device="cuda", generator=g) / D ** 0.5).to(dt)
    ex = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    p = torch.rand(T, k, device="cuda", generator=g) + 0.1 if weighted else None
    dy = torch.randn(*((T, O) if weighted else (T, k, O)), device="cuda", generator=g).to(dt)
    plan = X.plan_experts(ex, E)
    out = X.expert_linear(x, w, plan, p)
    dx, = torch.autograd.grad(out, x, dy)
    plan.check()
    out0, dx0 = _exact(x.detach(), w, ex, p, dy)
    if weighted:
        _one_rounding(out, out0)
    _one_rounding(dx, dx0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_large_terms_that_cancel(dt):
    """Two choices of weight 1000 and -1000 through matrices that differ by little: each term leaves the range of fp16 (up to
    3e5), their sum does not.  The terms carry fp32 errors of about 2^-22 of 3e5 (0.07) before they cancel; the sum's own
    rounding is up to half a step of its type."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T, D, O = 200, 64, 48
    x = torch.rand(T, D, device="cuda", generator=g).to(dt).requires_grad_()
    w0 = torch.rand(O, D, device="cuda", generator=g).to(dt) * 8
    w1 = w0.clone()
    w1[:, 0] += 0.25
    w = torch.stack([w0, w1])
    ex = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").expand(T, 2).contiguous()
    p = torch.tensor([[1000.0, -1000.0]], device="cuda").expand(T, 2).contiguous()
    dy = torch.rand(T, O, device="cuda", generator=g).to(dt)
    out = X.expert_linear(x, w, X.plan_experts(ex, 2), p)
    dx, = torch.autograd.grad(out, x, dy)
    out0, dx0 = _exact(x.detach(), w, ex, p, dy)
    u = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -11
    for got, want in ((out, out0), (dx, dx0)):
        assert torch.isfinite(got).all()
        assert ((got.detach().double() - want).abs() <= u * want.abs() + 0.5).all()
