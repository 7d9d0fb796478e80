"""Expert products on pairs of CTAs (cta_group::2), all forms that take them: forward, dx, dx with the gradient of the routing
weights, and the gradient of the matrices with and without weights, bf16 and fp16, with full 256-column tiles, narrower ones
(192 columns: 96 a CTA, one and a half swizzle atoms) and experts with an odd number of 128-row tiles or none.
Errors are bounded by the 2-norm of rounding the 64-bit result to the type (fp32 arithmetic adds 2 percent at most)."""
import pytest
import torch

from mace_onegpu import _native as N
from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu


def _near(got, want, slack=1.02):
    best = (want.to(got.dtype).double() - want).norm() if got.dtype != torch.float32 else 1e-6 * want.norm()
    mine = (got.double() - want).norm()
    assert mine <= slack * best, float(mine / best)


def _experts(T, E, g):
    """Uneven loads, an expert without slots, tokens without an expert."""
    ex = torch.randint(0, E, (T, 1), device="cuda", generator=g, dtype=torch.int32)
    if E > 2:
        ex[ex == 1] = 0
    ex[torch.rand(T, 1, device="cuda", generator=g) < 0.02] = -1
    return ex


# T, E, D, O: tiles of 256 rows times tiles of 256 columns are at least 8 for each of the 74 pairs
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,D,O", [(40_000, 3, 1088, 1024), (160_000, 4, 1024, 192), (54_000, 2, 1024, 700)])
def test_forward_on_pairs(T, E, D, O, dt):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, D, device="cuda", generator=g).to(dt)
    w = (torch.randn(E, O, D, device="cuda", generator=g) / D ** 0.5).to(dt)
    ex = _experts(T, E, g)
    plan = X.plan_experts(ex, E)
    p = torch.rand(T, 1, device="cuda", generator=g)
    out = X.expert_linear(x, w, plan, p)
    plan.check()
    for e in range(E):
        t = torch.nonzero(ex[:, 0] == e)[:, 0]
        if len(t):
            _near(out[t], p[t].double() * (x[t].double() @ w[e].double().T))
    assert not out[ex[:, 0] < 0].any()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,D,O", [(40_000, 3, 1024, 1088), (160_000, 4, 192, 1024), (54_000, 2, 700, 1024)])
@pytest.mark.parametrize("weighted", [False, True])
def test_dx_on_pairs(T, E, D, O, dt, weighted):
    g = torch.Generator(device="cuda").manual_seed(T + 1)
    x = torch.randn(T, D, device="cuda", generator=g).to(dt)
    w = (torch.randn(E, O, D, device="cuda", generator=g) / D ** 0.5).to(dt)
    ex = _experts(T, E, g)
    plan = X.plan_experts(ex, E)
    p = torch.rand(T, 1, device="cuda", generator=g) if weighted else None
    dy = torch.randn(T, O, device="cuda", generator=g).to(dt)
    dx, _, dp = N.ops().expert_linear_bwd(dy if weighted else dy[:, None], x, w, plan.experts, plan.words, p, True, False, weighted)
    plan.check()
    for e in range(E):
        t = torch.nonzero(ex[:, 0] == e)[:, 0]
        if len(t) == 0:
            continue
        back = dy[t].double() @ w[e].double()
        _near(dx[t], back if p is None else p[t].double() * back)
        if weighted:
            _near(dp[t, 0], (x[t].double() * back).sum(1))
    assert not dx[ex[:, 0] < 0].any()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,D,O", [(48_000, 40, 1024, 1024), (130_000, 100, 192, 2048), (70_000, 60, 700, 1000)])
@pytest.mark.parametrize("weighted", [False, True])
def test_dw_on_pairs(T, E, D, O, dt, weighted):
    g = torch.Generator(device="cuda").manual_seed(T + 2)
    x = torch.randn(T, D, device="cuda", generator=g).to(dt)
    w = torch.zeros(E, O, D, device="cuda", dtype=dt)
    ex = _experts(T, E, g)
    plan = X.plan_experts(ex, E)
    p = torch.rand(T, 1, device="cuda", generator=g) if weighted else None
    dy = torch.randn(T, O, device="cuda", generator=g).to(dt)
    _, dw, _ = N.ops().expert_linear_bwd(dy if weighted else dy[:, None], x, w, plan.experts, plan.words, p, False, True, False)
    plan.check()
    for e in range(E):
        t = torch.nonzero(ex[:, 0] == e)[:, 0]
        if len(t) == 0:
            assert not dw[e].any()
            continue
        z = dy[t].double() if p is None else p[t].double() * dy[t].double()
        _near(dw[e], z.T @ x[t].double())
