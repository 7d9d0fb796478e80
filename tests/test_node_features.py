"""ThreePassEngine.node_features hands out the features of the evaluation that has just run, or refuses."""
import pytest
import torch

from mace_onegpu import engine as E
from mace_onegpu import model as M
from mace_onegpu import neighbors, structures


class _Plan:
    nl = nt = 5


def test_refused_before_any_evaluation():
    eng = E.ThreePassEngine.__new__(E.ThreePassEngine)          # the host side only
    eng._buf, eng._features, eng.device = {}, None, torch.device("cpu")
    with pytest.raises(RuntimeError, match="last evaluation"):
        eng.node_features(_Plan())


def _plan(eng, n, seed, pinned=False):
    pos, Z, box = structures.water_box(n, seed=seed)
    cols = torch.as_tensor(structures.species_columns(Z, eng.model.arch.atomic_numbers))
    pi, pj, rij = (torch.as_tensor(t) for t in neighbors.neighbor_list(pos, box, eng.model.arch.r_max))
    if pinned:
        pi, pj, rij = pi.to(torch.int32).pin_memory(), pj.to(torch.int32).pin_memory(), rij.double().contiguous().pin_memory()
    return eng.plan(pi, pj, rij, cols, len(Z), len(Z))


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("pinned", [False, True])
def test_features_belong_to_the_last_evaluation(graph, pinned):
    mdl = M.default_model(0)
    cols = sorted(set(structures.species_columns(structures.water_box(2, seed=0)[1], mdl.arch.atomic_numbers).tolist()))
    eng = E.ThreePassEngine(mdl, cols, chunk=256, device="cuda")
    small, large = _plan(eng, 4, 1, pinned), _plan(eng, 5, 2, pinned)
    with pytest.raises(RuntimeError, match="last evaluation"):
        eng.node_features(small)
    got = {}
    for p in (small, large, small):                # the second evaluation makes the buffers larger
        eng.evaluate(p, graph=graph)
        h = eng.node_features(p)
        assert h.shape == (p.nt, 4, 128) and torch.isfinite(h).all() and h.any()
        if id(p) in got:
            assert (h - got[id(p)]).abs().max() <= 1e-5 * h.abs().max()
        got[id(p)] = h.clone()
        other = large if p is small else small
        with pytest.raises(RuntimeError, match="last evaluation"):
            eng.node_features(other)
    fresh = E.ThreePassEngine(mdl, cols, chunk=256, device="cuda")
    plain = _plan(fresh, 5, 2)
    fresh.evaluate(plain)
    h = fresh.node_features(plain)
    assert (h - got[id(large)]).abs().max() <= 1e-5 * h.abs().max()
