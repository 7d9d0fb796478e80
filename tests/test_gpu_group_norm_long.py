"""Group norm of many short samples and one that is thousands of times as long: samples are cut by their mean length, so a thread of the
long one adds 30,000 to 140,000 rows, in runs of 512.

The long sample's rows are 0 first (a thread's own first row, which its sums are relative to) and then 0.1 and 0.3 in turns of 64
rows, and dy is 0.1: sums of like values, where an addition loses the same part of an ulp each time.  Added in one go 137,500
values of 0.1 come out 0.12% low (bfloat16's 0.1: 0.20%) and their squares 0.13%.

Tolerances.  Of R rows of a thread no sum is off by more than e = (512 + R / 512) 2^-25 of itself, 2.3e-5 for 137,500; the joins over
threads add (8 + log2 M) 2^-24.  Mean 0.2, variance 0.01, mean square 0.05: x - mean is off by 0.2 e, two standard deviations of it, and
the variance by (0.05 + 2 0.04) e, 13 times itself, so that xh (at most 2 in size) is off by (2 + 13) e, 3.5e-4 at most.  a = dy has no
part that is left in dx: dx is what mean(a) and mean(a xh) are off by, r 0.1 (e + 2 e + the roundings of xh): 10 x 0.1 x 1e-4."""
import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
E32, EPS = 2.0 ** -23, 1e-5
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


# one launch (a CTA a sample), several launches with few parts a sample, one group wider than a pass of a CTA's threads
@pytest.mark.parametrize("dt,c,groups,n,short,long,where", [
    (torch.bfloat16, 128, 8, 20000, 60, 1_100_000, 7), (torch.float32, 128, 8, 20000, 30, 550_000, 20000),
    (torch.bfloat16, 128, 8, 200, 500, 2_000_000, 100), (torch.float32, 128, 8, 300, 300, 1_500_000, 0),
    (torch.float32, 4096, 1, 300, 3, 6000, 150), (torch.bfloat16, 8192, 1, 300, 3, 6000, 2),
    (torch.bfloat16, 15, 3, 20000, 30, 600_000, 9), (torch.float32, 36, 2, 5000, 100, 900_001, 5000)])
def test_one_long_sample(dt, c, groups, n, short, long, where):
    g = torch.Generator(device="cuda").manual_seed(n)
    lens = torch.full((n + 1,), short)
    lens[where] = long
    off = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(lens, 0)])
    lo, hi = int(off[where]), int(off[where + 1])
    x = torch.randn(int(off[-1]), c, device="cuda", generator=g).to(dt)
    turn = torch.arange(long, device="cuda") // 64
    x[lo:hi] = torch.where(turn == 0, 0.0, torch.where(turn % 2 == 0, 0.1, 0.3)).to(dt)[:, None]
    w, b = torch.ones(c, device="cuda", requires_grad=True), torch.zeros(c, device="cuda", requires_grad=True)
    dy = torch.full_like(x, 0.1)
    xd = x.clone().requires_grad_()
    y = X.group_norm(xd, groups, w, b, eps=EPS, offsets=off.cuda())
    dx, dw, db = torch.autograd.grad(y, (xd, w, b), dy)
    v = x[lo:hi].double()                                     # all channels are alike: one group's statistics for all
    mean, var = v.mean(), v.var(unbiased=False)
    want = (v - mean) / (var + EPS).sqrt()
    assert bool(((y.detach()[lo:hi].double() - want).abs() <= U[dt] * want.abs() + 4e-4).all())
    assert float(dx[lo:hi].abs().max()) <= 1e-4
    total = float(dy[0, 0].double()) * int(off[-1])
    assert float((db.double() - total).abs().max()) <= 1e-4 * total
    # a sample's sum of xh is 0 over the channels of a group (not in each of them: the short samples' rows are random)
    assert float(dw.view(groups, -1).sum(1).abs().max()) <= 1e-4 * total * c / groups
    # the short samples are those of a call of their own, in another order of sums
    keep = torch.cat([x[:lo], x[hi:]])
    alone = X.group_norm(keep, groups, w, b, eps=EPS, offsets=torch.arange(n + 1).mul(short).cuda()).detach().double()
    rest = torch.cat([y[:lo], y[hi:]]).detach().double()
    assert bool(((rest - alone).abs() <= 2 * U[dt] * alone.abs() + 64 * E32).all())
