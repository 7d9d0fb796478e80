"""A product that gave up waiting (one load withheld, waits of 20 ms) leaves NaN where it has no result: nothing that could be
taken for one, whether anybody asks for the status or not."""
import pytest
import torch

from mace_onegpu import _native as N
from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu


@pytest.fixture
def withheld():
    N.check(N.lib().mace_b200_expert_test_hooks(20_000_000, 1), "expert_test_hooks")
    yield
    torch.cuda.synchronize()
    N.check(N.lib().mace_b200_expert_test_hooks(2_000_000_000, 0), "expert_test_hooks")


def _inputs(T, k, E, D, O, dt):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, D, device="cuda", generator=g).to(dt)
    w = (torch.randn(E, O, D, device="cuda", generator=g) / D ** 0.5).to(dt)
    ex = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    p = torch.rand(T, k, device="cuda", generator=g)
    dy = torch.randn(T, O, device="cuda", generator=g).to(dt)
    return x, w, X.plan_experts(ex, E), p, dy


def _right_or_nan(got, want):
    bad = torch.isnan(got)
    assert bad.any()
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dt,T,k,E,D,O", [(dt, *s) for dt in (torch.float32, torch.bfloat16, torch.float16)
                                           for s in ((300, 1, 1, 64, 64), (700, 2, 3, 128, 200), (40000, 1, 1, 1024, 1024))
                                           if dt != torch.float32 or s[0] < 40000])      # the last on pairs of CTAs
@pytest.mark.parametrize("need", ["out", "dx", "dw", "dx dweights"])
def test_a_product_that_gave_up_is_nan(dt, T, k, E, D, O, need, withheld):
    x, w, plan, p, dy = _inputs(T, k, E, D, O, dt)
    words = plan.words

    def run():
        if need == "out":
            return [N.ops().expert_linear(x, w, plan.experts, words, p)]
        r = N.ops().expert_linear_bwd(dy, x, w, plan.experts, words, p, "dx" in need, "dw" == need, "dweights" in need)
        return [t for t, n in zip(r, ("dx" in need, "dw" == need, "dweights" in need)) if n]

    got = run()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="gave up waiting"):
        plan.check()
    N.check(N.lib().mace_b200_expert_test_hooks(2_000_000_000, 0), "expert_test_hooks")
    for a, b in zip(got, run()):
        _right_or_nan(a, b)
