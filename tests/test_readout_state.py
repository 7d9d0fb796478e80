"""Host side of what the readout modules and Muon keep: types of state, refusals that come before any of it changes."""
import concurrent.futures
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mace_onegpu import optim


def test_loaded_state_of_narrow_parameters_stays_float32():
    p = torch.nn.Parameter(torch.zeros(4, 6, dtype=torch.bfloat16))
    saved = optim.Muon([p]).state_dict()
    state = {k: torch.rand(4, 6) for k in ("momentum_buffer", "rounding")}
    saved["state"] = {0: state}
    opt = optim.Muon([p])
    opt.load_state_dict(saved)
    for k, v in state.items():
        assert opt.state[p][k].dtype == torch.float32 and torch.equal(opt.state[p][k], v) and opt.state[p][k] is not v
    saved["state"][0]["momentum_buffer"] = state["momentum_buffer"].bfloat16()    # of a float32 checkpoint cast to 16 bits
    opt.load_state_dict(saved)
    assert opt.state[p]["momentum_buffer"].dtype == torch.float32


def _matrix(dt=torch.float32):
    return torch.nn.Parameter(torch.ones(4, 6, dtype=dt))


BAD = [dict(lr=-1.0), dict(lr=float("nan")), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0), dict(steps=17),
       dict(coefficients=(9.0, 0.0, 0.0)), dict(coefficients=((1.5, -0.5, 0.0),) * 4), dict(coefficients=(float("nan"), 0.0, 0.0)),
       dict(eps=0.0)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_muon_refuses_a_groups_own_values(bad):
    """In the constructor, in a group of its own, and where a group was edited: before any state is there."""
    with pytest.raises(ValueError):
        optim.Muon([_matrix()], **bad)
    with pytest.raises(ValueError):
        optim.Muon([dict(params=[_matrix()]), dict(params=[_matrix()], **bad)])
    p = _matrix()
    opt = optim.Muon([p])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[_matrix()], **bad))
    assert len(opt.param_groups) == 1
    p.grad = torch.ones_like(p)
    opt.param_groups[0].update(bad)
    with pytest.raises(ValueError):
        opt.step()
    assert not opt.state and torch.equal(p.detach(), torch.ones(4, 6))


def test_muon_refuses_parameters_before_state_changes():
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        optim.Muon([_matrix(torch.float64)])
    with pytest.raises(ValueError, match="matrices"):
        optim.Muon([_matrix(), torch.nn.Parameter(torch.zeros(3))])
    for shape in ((1, 65537), (65537, 1), (256, 256, 1, 1)):
        with pytest.raises(ValueError, match="at most"):
            optim.Muon([torch.nn.Parameter(torch.zeros(shape))])
    p = _matrix()
    opt = optim.Muon([p])
    opt.step()                                                 # without a gradient there is nothing to do
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="CUDA"):
        opt.step()
    assert not opt.state


def test_coefficient_tables_from_many_threads():
    """More tables than are kept, made by threads at once: each call gets its own values."""
    wrong = []

    def work(seed):
        for i in range(2000):
            a = 1.0 + ((seed * 977 + i * 31) % 200) / 1000
            t = optim._table(3, (a, -0.5, 0.0))
            if t.shape != (3, 3) or float(t[2, 0]) != a:
                wrong.append(a)

    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        with concurrent.futures.ThreadPoolExecutor(8) as pool:
            for f in [pool.submit(work, s) for s in range(8)]:
                f.result()                                     # a KeyError of a thread comes back here
    finally:
        sys.setswitchinterval(before)
    assert not wrong


def test_polynomials_seen_without_values_are_looked_at_later():
    """Under FakeTensorMode a table has no values: what is refused is still refused afterwards."""
    bad = dict(coefficients=(8.5, 0.25, 0.0))
    with FakeTensorMode():
        optim.Muon([_matrix()], **bad)
    with pytest.raises(ValueError, match="reaches"):
        optim.Muon([_matrix()], **bad)
