"""Host side of layer norm, expert routing and expert products: argument checks of the C ABI and the Python module that
come before any launch, and the plain fp64 forms the GPU tests compare with, against torch's own operations."""
import math

import pytest
import torch

import expert_refs as R
from mace_onegpu import _native as N
from mace_onegpu import experts as X


def test_plan_size_and_refusals():
    L, n = N.lib(), N.c_i64()
    assert L.mace_b200_expert_plan_words(1000, 7, N.byref(n)) == 0 and n.value > 1000
    small = n.value
    assert L.mace_b200_expert_plan_words(2000, 7, N.byref(n)) == 0 and n.value > small
    for slots, E in ((-1, 4), (10, 0), (10, 1025), (2 ** 29 + 1, 4)):
        assert L.mace_b200_expert_plan_words(slots, E, N.byref(n)) < 0
        assert b"bad sizes" in L.mace_b200_last_error()


def test_bad_arguments_come_back_as_codes():
    L, n = N.lib(), N.c_i64()
    assert L.mace_b200_layer_norm_bwd_workspace(10, 0, N.byref(n)) < 0 and b"width 0" in L.mace_b200_last_error()
    assert L.mace_b200_layer_norm_fwd(None, 4, None, None, None, None, None, 3, 8, 1e-5, 0, 0, None) < 0
    assert b"row stride 4" in L.mace_b200_last_error()
    assert L.mace_b200_layer_norm_fwd(None, 8, None, None, None, None, None, 3, 8, 1e-5, 9, 9, None) < 0
    assert b"unsupported types" in L.mace_b200_last_error()
    assert L.mace_b200_route_fwd(None, 600, None, None, None, 3, 600, 2, 1, 1, 1, 1, 1.0, 0, None) < 0
    assert b"at most 512 experts" in L.mace_b200_last_error()
    assert L.mace_b200_expert_linear_workspace(10, 2, 4, 0, 8, 0, 0, 1, 0, N.byref(n)) < 0
    assert b"bad sizes" in L.mace_b200_last_error()


def test_module_checks_arguments():
    with pytest.raises(ValueError, match="softmax"):
        X.route(torch.zeros(2, 4), 1, score="relu")
    with pytest.raises(ValueError, match="integer"):
        X.plan_experts(torch.zeros(2, 2), 4)
    with pytest.raises(ValueError, match="positive"):
        X.plan_experts(torch.zeros(2, 2, dtype=torch.int64), 0)
    plan = X.plan_experts(torch.zeros(3, dtype=torch.int64), 4)
    assert plan.experts.shape == (3, 1) and plan.experts.dtype == torch.int32
    wide = X.plan_experts(torch.tensor([[0, 2 ** 32 + 1], [-1, 3]]), 3)     # never wraps into the range
    assert wide.experts.tolist() == [[0, -2], [-1, -2]]
    with pytest.raises(TypeError, match="ExpertPlan"):
        X.expert_linear(torch.zeros(3, 8), torch.zeros(4, 8, 8), plan.experts)
    with pytest.raises(ValueError, match="w must be"):
        X.expert_linear(torch.zeros(3, 8), torch.zeros(5, 8, 8), plan)


def test_shape_functions():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = N.ops()
    with FakeTensorMode():
        x = torch.empty(6, 16, device="cuda")
        assert ops.layer_norm(x, None, None, 1e-5).shape == (6, 16)
        w, e = ops.route(torch.empty(6, 8, device="cuda", dtype=torch.bfloat16), None, 2, True, 1, 1, True, 1.0)
        assert w.shape == e.shape == (6, 2) and w.dtype == torch.float32 and e.dtype == torch.int32
        m = torch.empty(8, 5, 16, device="cuda")
        assert ops.expert_linear(x, m, e, None, w).shape == (6, 5)
        assert ops.expert_linear(x, m, e, None, None).shape == (6, 2, 5)
        y, mean, rstd = ops.layer_norm_fwd(x, None, None, 1e-5)
        assert [t.shape for t in ops.layer_norm_bwd(y, x, None, mean, rstd, True, True, True, False)] == [(6, 16), (16,), (16,)]
        plan = ops.expert_plan(e, 8)
        dx, dm, dw = ops.expert_linear_bwd(torch.empty(6, 5, device="cuda"), x, m, e, plan, w, True, True, True)
        assert dx.shape == x.shape and dm.shape == m.shape and dw.shape == w.shape
        assert ops.route_bwd(w, torch.empty(6, 8, device="cuda"), e, True, True, 1.0).shape == (6, 8)


def test_plain_layer_norm_is_torchs():
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((7, 33), (33,), (33,), (7, 33)))
    ins = [t.requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5)
    want = (y, *torch.autograd.grad(y, ins, dy))
    for a, c in zip(R.layer_norm(*[t.detach() for t in ins], 1e-5, dy), want):
        assert (a - c).abs().max() < 1e-12


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_plain_route_is_torchs(score, renorm):
    g = torch.Generator().manual_seed(1)
    l = torch.randn(20, 12, generator=g, dtype=torch.float64)
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    top = torch.topk(l, 4, dim=1).indices
    w = s.gather(1, top)
    w = w / w.sum(1, keepdim=True) if renorm else w
    W, E, _ = R.route(l, 4, score=score, renormalize=renorm)
    assert torch.equal(E, top) and (W - w).abs().max() < 1e-12
    assert (R.route_weights(l, E, score, renorm) - w).abs().max() < 1e-12
    # groups: the two best of each of 3, two groups stay
    W, E, _ = R.route(l, 2, score="sigmoid", groups=3, top_groups=2)
    val = torch.sort(torch.sigmoid(l).view(20, 3, 4), dim=2, descending=True).values[..., :2].sum(2)
    worst = val.argmin(1)
    assert not (E // 4 == worst[:, None]).any()
    W, E, _ = R.route(torch.full((1, 3), -math.inf), 2)
    assert E.tolist() == [[-1, -1]] and not W.any()


def test_plain_products_are_torchs():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 5, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(3, 4, 5, generator=g, dtype=torch.float64, requires_grad=True)
    p = torch.rand(9, 2, generator=g, dtype=torch.float64, requires_grad=True)
    ex = torch.randint(0, 3, (9, 2), generator=g)
    dy = torch.randn(9, 4, generator=g, dtype=torch.float64)
    z = torch.einsum("tkod,td->tko", w[ex], x)
    out = (p[..., None] * z).sum(1)
    want = (out, *torch.autograd.grad(out, (x, w, p), dy))
    got = R.expert_linear(x.detach(), w.detach(), ex, p.detach(), dy)
    for a, b in zip(got, want):
        assert (a[0] - b).abs().max() < 1e-12 and (a[1] >= a[0].abs() - 1e-12).all()
