"""Every term of group norm's gradients in every form of the kernels, by the check of group_norm_checks.py (which test_group_norm_checks.py
shows to reject the formulas without them): one launch, several launches (asked of the workspace's size), ragged, wide groups."""
import pytest
import torch

import group_norm_checks as C
from mace_onegpu import _native as N
from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _streams(rows, n, length, c, groups, ragged, dt):
    """Whether the forward pass takes several launches (it then needs sums in the workspace); the backward pass, which holds twice the
    bytes, does so, too."""
    f = N.c_i64()
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt]
    assert N.lib().mace_b200_group_norm_workspace(rows, n, length, c, groups, ragged, code, 0, N.byref(f)) == 0
    return f.value > 0


def _check(rows, c, groups, edges, dt, act, shape=None):
    x, w, b, dy = C.inputs(rows, c, groups, edges, dt, rows + c, "cuda")
    off = None if shape else torch.tensor(edges).cuda()
    xd, wd, bd = (t.clone().requires_grad_() for t in (x.view(shape) if shape else x, w, b))
    y = X.group_norm(xd, groups, wd, bd, eps=C.EPS, activation=act, offsets=off)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.view(xd.shape))
    assert C.failures(x, groups, w, b, dy, act, edges, dt, y.detach().view(rows, c), dx.view(rows, c), dw, db) == []


@pytest.mark.parametrize("dt,n,l,c,groups", [("f32", 1, 192, 128, 8), ("bf16", 2, 9, 4104, 4), ("f16", 5, 64, 15, 3), ("f32", 2, 40, 8192, 2), ("f32", 3, 20, 96, 32),
                                             ("bf16", 40, 70, 128, 8)])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_one_launch(dt, n, l, c, groups, act):
    assert not _streams(n * l, n, l, c, groups, 0, DT[dt])
    _check(n * l, c, groups, [i * l for i in range(n + 1)], DT[dt], act, (n, l, c))


@pytest.mark.parametrize("dt,n,l,c,groups", [("f32", 3, 300, 4096, 1), ("bf16", 2, 700, 8200, 2), ("f16", 2, 1501, 1030, 2), ("bf16", 700, 33, 1024, 4),
                                             ("f32", 9, 6000, 36, 12), ("bf16", 1, 45, 70000, 7), ("f32", 1, 24000, 128, 8), ("f16", 64, 500, 128, 8),
                                             ("f32", 2, 300_001, 8, 1)])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_several_launches(dt, n, l, c, groups, act):
    assert _streams(n * l, n, l, c, groups, 0, DT[dt])
    _check(n * l, c, groups, [i * l for i in range(n + 1)], DT[dt], act, (n, l, c))


@pytest.mark.parametrize("dt,edges,rows,c,groups,several", [
    ("f32", [0, 100, 60000], 60000, 256, 4, True), ("bf16", [0, 100, 150000], 150000, 256, 32, True), ("f16", [7, 7, 20000, 40000], 40001, 264, 3, True),
    ("bf16", [3, 3, 4, 4, 40, 300, 301, 301], 310, 128, 8, False), ("f32", list(range(2, 9003, 9)), 9003, 64, 8, False)])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_ragged(dt, edges, rows, c, groups, several, act):
    assert _streams(rows, len(edges) - 1, 0, c, groups, 1, DT[dt]) == several
    _check(rows, c, groups, edges, DT[dt], act)
