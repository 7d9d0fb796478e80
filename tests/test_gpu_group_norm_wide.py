"""Group norm of rows of millions of channels: more column blocks than a grid has, and no more parts (each with sums of every column
in the backward pass) than rows."""
import pytest
import torch

from mace_onegpu import _native as N
from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.mark.parametrize("l,c,groups", [(2, 2 ** 27, 2 ** 17), (3, 2 ** 22, 2 ** 10), (64, 2 ** 20, 8)])
def test_wide_rows(l, c, groups):
    """Tolerances: groups of 2,048 to 8 million values of size one: statistics to (8 + 23) 2^-23 (see test_gpu_group_norm.py), results up to 6
    rounded to bfloat16 (2^-8), gradients of sums of up to 64 rows."""
    g = torch.Generator(device="cuda").manual_seed(c)
    cg = c // groups
    x = torch.empty(1, l, c, device="cuda", dtype=torch.bfloat16).normal_(generator=g).requires_grad_()
    dy = torch.empty(1, l, c, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    w = torch.empty(c, device="cuda", dtype=torch.bfloat16).normal_(generator=g).requires_grad_()
    y = X.group_norm(x, groups, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for k in {0, groups // 2, groups - 1}:
        at = slice(k * cg, (k + 1) * cg)
        v, d, u = x.detach()[0, :, at].double(), dy[0, :, at].double(), w.detach()[at].double()
        r = 1 / (v.var(unbiased=False) + EPS).sqrt()
        xh = (v - v.mean()) * r
        a = d * u
        for got, want in ((y.detach()[0, :, at], xh * u), (dx[0, :, at], r * (a - a.mean() - xh * (a * xh).mean())), (dw[at], (d * xh).sum(0))):
            assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * max(1.0, float(want.abs().max()))).all())


def test_workspace_of_wide_rows():
    """Sums of every column for each row at most."""
    n = N.c_i64()
    for rows, c in ((64, 2 ** 20), (2, 2 ** 27), (3, 2 ** 22)):
        assert N.lib().mace_b200_group_norm_workspace(rows, 1, rows, c, 8, 0, 1, 1, N.byref(n)) == 0
        assert n.value <= 2 * c * rows + (3 * rows + 2) * 8
