"""Muon of bfloat16 and float16 parameters: its state is float32, and updates and decays below half a step of the type add up.

Tolerances.  A parameter is its float32 value rounded once (half a step, U).  The float32 recurrence rounds twice a step: 2^-23 of the
value.  An update is compared with the U = orthogonalize(..) of gradients that differ by float32 roundings: its scale differs by an ulp,
so each rounding within it (operands to float16, the result to bfloat16) may fall the other way, and the two are each off by up to TOL =
7.6e-3 of the norm (the bound that test_gpu_orth.py derives), not of each element: 2 TOL of the norms of the updates."""
import copy

import pytest
import torch

from mace_onegpu import optim as X

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TOL = 2.0 ** -8 + 15 * 2.0 ** -11 / 2


def _param(dt, *shape, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.nn.Parameter((0.2 * torch.randn(*shape, device="cuda", generator=g)).to(dt))


@pytest.mark.parametrize("dt,lr,decay", [(torch.bfloat16, 0.02, 0.05), (torch.float16, 0.02, 0.01), (torch.float32, 0.02, 0.05)])
def test_small_decays_add_up(dt, lr, decay):
    """1 - lr decay lies within half a step of one: rounded each time, no parameter would change.  Without a gradient U is 0."""
    p = _param(dt, 40, 25)
    before = p.detach().double()
    opt = X.Muon([p], lr=lr, weight_decay=decay)
    p.grad = torch.zeros_like(p)
    for _ in range(1000):
        opt.step()
    want = before * (1 - lr * decay) ** 1000
    # float16: half of its smallest value, too
    assert bool(((p.detach().double() - want).abs() <= (U[dt] + 2000 * 2.0 ** -24) * want.abs() + 2.0 ** -25).all())


@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_small_updates_add_up(dt, nesterov):
    p = _param(dt, 3, 33, 20)
    ref, v = p.detach().double(), torch.zeros(3, 33, 20, device="cuda", dtype=torch.float64)
    opt = X.Muon([p], lr=2e-4, momentum=0.9, nesterov=nesterov)
    p.grad = _param(dt, 3, 33, 20, seed=1).detach()
    way = 0.0
    for _ in range(300):
        v = 0.9 * v + p.grad.double()
        d = p.grad.double() + 0.9 * v if nesterov else v
        up = 2e-4 * (33 / 20) ** 0.5 * X.orthogonalize(d.float()).double()
        ref, way = ref - up, way + float(up.norm())
        opt.step()
    assert opt.state[p]["momentum_buffer"].dtype == opt.state[p]["rounding"].dtype == torch.float32
    tol = ((U[dt] + 600 * 2.0 ** -24) * ref.abs() + 2.0 ** -25).norm() + 2 * TOL * way
    assert float((p.detach().double() - ref).norm()) <= float(tol)
    assert way > 5 * float(tol)                               # (no step alone changes most of the values)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_saved_state_goes_on_alike(dt):
    p, q = _param(dt, 64, 48), None
    opt = X.Muon([p], lr=1e-3, weight_decay=0.01)
    grads = [_param(dt, 64, 48, seed=s).detach() for s in range(10)]
    for i, g in enumerate(grads):
        if i == 5:
            q = torch.nn.Parameter(p.detach().clone())
            saved = copy.deepcopy(opt.state_dict())
            other = X.Muon([q], lr=1e-3, weight_decay=0.01)
            other.load_state_dict(saved)
        for o, t in ((opt, p), (other, q)) if i >= 5 else ((opt, p),):
            t.grad = g
            o.step()
    assert torch.equal(p, q)
    for key, value in opt.state[p].items():
        assert torch.equal(value, other.state[q][key]) and value.dtype == torch.float32
    saved["state"][0]["momentum_buffer"].fill_(7)              # and is a copy
    assert not (other.state[q]["momentum_buffer"] == 7).any()


def test_a_parameter_set_from_outside_stays_set():
    p = _param(torch.bfloat16, 32, 32)
    opt = X.Muon([p], lr=1e-3)
    p.grad = _param(torch.bfloat16, 32, 32, seed=1).detach()
    opt.step()
    with torch.no_grad():
        p.fill_(3.0)
    p.grad = torch.zeros_like(p)
    opt.param_groups[0].update(lr=0.0)
    opt.step()
    assert bool((p == 3.0).all())
