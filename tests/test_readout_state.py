"""Host side of what the readout modules and Muon keep: types of state, refusals that come before any of it changes."""
import concurrent.futures
import sys

import torch

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
