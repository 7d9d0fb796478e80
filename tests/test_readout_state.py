"""Host side of what the readout modules and Muon keep: types of state, refusals that come before any of it changes."""
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
