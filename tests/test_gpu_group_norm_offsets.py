"""Group norm over offsets that do not ascend: samples could share rows, so every row of the result and of dx is NaN, in each form of
the kernels (one launch, several launches, the offsets looked through by a launch of their own) and in every run; offsets that only
leave the rows make their own samples NaN."""
import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu


def _both(x, off, groups, act="silu"):
    xd = x.clone().requires_grad_()
    w = torch.ones(x.shape[1], device="cuda", dtype=x.dtype, requires_grad=True)
    y = X.group_norm(xd, groups, w, activation=act, offsets=off)
    dx, dw = torch.autograd.grad(y, (xd, w), torch.ones_like(y))
    return y.detach(), dx, dw


OFFSETS = {
    "samples 0 and 3 share rows 40 to 49": [0, 50, 30, 40, 100],
    "rows before the first and of a sample": [20, 10, 60],
    "rows behind the last and of a sample": [0, 90, 30],
    "the last one descends": [0, 100, 99],
    "behind the rows and back": [0, 300, 200, 50, 100],
    "before the rows and back": [5, -5, 100],
}


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("name", sorted(OFFSETS))
def test_every_row_is_nan(name, index, act):
    x, off = torch.randn(100, 32, device="cuda"), torch.tensor(OFFSETS[name], dtype=index).cuda()
    for _ in range(10):
        y, dx, dw = _both(x, off, 4, act)
        assert y.isnan().all() and dx.isnan().all() and dw.isnan().all()


@pytest.mark.parametrize("rows,c,n", [(60000, 128, 3), (60000, 128, 1024), (60000, 128, 1025), (60000, 64, 5000), (9000, 32, 9000),
                                      (200000, 32, 180000)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_one_step_back_among_many(rows, c, n, dt):
    """In the several-launch form, and with more samples than a CTA looks at."""
    x = torch.randn(rows, c, device="cuda").to(dt)
    good = torch.linspace(0, rows, n + 1).long()
    y, dx, dw = _both(x, good.cuda(), 4)
    assert y.isfinite().all() and dx.isfinite().all() and dw.isfinite().all()
    for at in (0, n // 2, n - 1):
        off = good.clone()
        off[at] = off[at + 1] + 1
        y, dx, dw = _both(x, off.cuda(), 4)
        assert y.isnan().all() and dx.isnan().all() and dw.isnan().all()
        assert torch.equal(X.group_norm(x, 4, offsets=off.cuda()).isnan(), torch.ones_like(x, dtype=torch.bool))


@pytest.mark.parametrize("n", [4, 3000])
def test_offsets_that_leave_the_rows(n):
    x = torch.randn(6000, 32, device="cuda")
    good = torch.linspace(0, 6000, n + 1).long()
    want, wdx, _ = _both(x, good.cuda(), 4)
    off = good.clone()
    off[0], off[-1] = -3, 7000
    y, dx, _ = _both(x, off.cuda(), 4)
    lo, hi = int(good[1]), int(good[-2])
    for got, ref in ((y, want), (dx, wdx)):
        assert got[:lo].isnan().all() and got[hi:].isnan().all()
        assert torch.equal(got[lo:hi], ref[lo:hi])


def test_a_replay_sees_new_offsets():
    x = torch.randn(8000, 32, device="cuda")
    off = torch.linspace(0, 8000, 2001).long().cuda()
    want = X.group_norm(x, 4, offsets=off)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = X.group_norm(x, 4, offsets=off)
    for bad in (False, True, False):
        if bad:
            off[1000] += 100
        g.replay()
        torch.cuda.synchronize()
        assert held.isnan().all() if bad else torch.equal(held, want)
        if bad:
            off[1000] -= 100
