"""Group norm with an activation (mace_onegpu.readout.group_norm) against the plain fp64 form of tests/readout_refs.py: types,
odd group widths, strides, single rows, ragged and empty samples, rows of no sample, several samples to a CTA, samples that do not
fit on the chip, large means, non-finite values, streams, graphs, and gradients against the formula's and against differences.

Tolerances.  u(type) is the largest relative error of one rounding: 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32).  The statistics
are fp32 sums over M values (pairwise over threads, at most a few hundred in a row): x - mean is off by (8 + log2 M) 2^-23 of the
largest |x - mean| and one ulp of |x|, which r = 1 / std scales; an activation's slope is at most 1.13 and the change of its slope at
most 0.8, so z's error reaches y and f' at most about once.  dx adds a mean over M of products of a few of those."""
import math

import pytest
import torch

import readout_refs as R
from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E32 = 2.0 ** -23
EPS = 1e-5


def _data(rows, c, dt, seed, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=g) * 2 + mean * torch.randn(c, generator=g)).to(dt)
    w = (1 + 0.3 * torch.randn(c, generator=g)).to(dt)
    b = (0.3 * torch.randn(c, generator=g)).to(dt)
    return x, w, b, torch.randn(rows, c, generator=g).to(dt)


def _stats(x, groups, edges):
    """1 / std and the largest |x| of each row's group, and how far x - mean can be off, as [rows, C]."""
    rows, c = x.shape
    r, top, m = torch.ones(rows, c, dtype=torch.float64), torch.zeros(rows, c, dtype=torch.float64), 1
    for lo, hi in zip(edges, edges[1:]):
        if hi > lo:
            v = x[lo:hi].double().reshape(hi - lo, groups, -1)
            sd = (v.var((0, 2), unbiased=False, keepdim=True) + EPS).sqrt()
            r[lo:hi] = (1 / sd).expand_as(v).reshape(hi - lo, c)
            top[lo:hi] = v.abs().amax((0, 2), keepdim=True).expand_as(v).reshape(hi - lo, c)
            m = max(m, v[:, 0].numel())
    return r, top, (8 + math.log2(m)) * E32


def _close(got, want, tol, dt, what):
    assert got.dtype == dt and got.shape == want.shape
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= U[dt] * want.abs() + tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol)[bad].max())}"


def _check(x, groups, w, b, dy, act, edges, dt, y, dx, dw, db):
    y0, dx0, dw0, db0 = R.group_norm_grads(x, groups, w, b, EPS, act, edges, dy)
    r, top, e = _stats(x, groups, edges)
    off = e * (1 + r * top)                                   # of xh
    wmax, bmax, dmax = float(w.abs().max()), float(b.abs().max()), float(dy.abs().max())
    xh = float((r * top).max()) * 2
    _close(y, y0, 2 * off * wmax + 8 * E32 * (xh * wmax + bmax), dt, "y")
    slope = 1 + wmax * (1 + xh)                               # of a = dy f'(z) w and of a xh in xh
    tol = 8 * off.max() * r * dmax * wmax * slope * (1 + xh)
    _close(dx, dx0, tol, dt, "dx")
    n = x.shape[0]
    tol = float(off.max()) * dmax * slope * n + (8 + math.log2(n + 1)) * E32 * dmax * (1 + xh) * n ** 0.5 * 8
    _close(dw, dw0, tol, dt, "dw")
    _close(db, db0, tol, dt, "db")


def _run(x, groups, w, b, dy, act, dt, shape=None, offsets=None):
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x if shape is None else x.view(shape), w, b))
    y = X.group_norm(xd, groups, wd, bd, eps=EPS, activation=act, offsets=offsets)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.cuda().view(xd.shape))
    assert torch.equal(y.detach(), X.group_norm(xd.detach(), groups, wd.detach(), bd.detach(), eps=EPS, activation=act,
                                                offsets=offsets))
    y2 = X.group_norm(xd, groups, wd, bd, eps=EPS, activation=act, offsets=offsets)
    again = torch.autograd.grad(y2, (xd, wd, bd), dy.cuda().view(xd.shape))
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))     # fixed order of the sums
    c = x.shape[1]
    return y.detach().reshape(-1, c), dx.reshape(-1, c), dw, db


def _clear_of_kinks(x, groups, w, b, edges, act):
    """relu's slope jumps at 0: inputs whose z are all further from it than any error of z."""
    z = R.group_norm(x.double(), groups, w.double(), b.double(), EPS, None, edges)
    return act != "relu" or float(z.abs().min()) > 2e-5


SHAPES = [(1, 1, 8, 1), (1, 1, 128, 8), (3, 1, 96, 32), (1, 7, 24, 8), (2, 5, 30, 2), (4, 33, 128, 8), (1, 192, 128, 8),
          (5, 64, 15, 3), (2, 50, 520, 4), (1, 20, 2048, 1), (2, 9, 4100, 4), (3, 17, 64, 64), (2, 40, 8192, 2), (1, 3, 20000, 1)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,l,c,groups", SHAPES)
def test_dense(n, l, c, groups, dt):
    dt, act = DT[dt], [None, "silu", "gelu"][(n + l + c) % 3]
    x, w, b, dy = _data(n * l, c, dt, n + l + c)
    edges = [i * l for i in range(n + 1)]
    y, dx, dw, db = _run(x, groups, w, b, dy, act, dt, (n, l, c))
    if l * c // groups == 1:                                  # x is its own mean
        assert not dx.any()
        return
    _check(x, groups, w, b, dy, act, edges, dt, y, dx, dw, db)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_activations(act, dt):
    dt = DT[dt]
    for seed in range(100):                                   # chosen by the inputs alone
        x, w, b, dy = _data(60, 32, dt, seed)
        if _clear_of_kinks(x, 4, w, b, [0, 20, 40, 60], act):
            break
    y, dx, dw, db = _run(x, 4, w, b, dy, act, dt, (3, 20, 32))
    _check(x, 4, w, b, dy, act, [0, 20, 40, 60], dt, y, dx, dw, db)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("c,groups", [(128, 8), (36, 4), (15, 5), (512, 32)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_ragged(c, groups, dt, index):
    """Empty samples first, between and last, single rows, rows before the first and behind the last sample."""
    dt = DT[dt]
    edges = [3, 3, 4, 4, 40, 300, 301, 301]
    x, w, b, dy = _data(310, c, dt, c)
    y, dx, dw, db = _run(x, groups, w, b, dy, "silu", dt, None, torch.tensor(edges, dtype=index).cuda())
    assert not y[:3].any() and not y[301:].any() and not dx[:3].any() and not dx[301:].any()
    _check(x, groups, w, b, dy, "silu", edges, dt, y, dx, dw, db)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_many_small_samples(dt):
    """More samples than CTAs: each CTA goes over several."""
    dt = DT[dt]
    lens = torch.randint(0, 9, (5000,), generator=torch.Generator().manual_seed(0))
    edges = [0, *torch.cumsum(lens, 0).tolist()]
    x, w, b, dy = _data(edges[-1], 32, dt, 3)
    y, dx, dw, db = _run(x, 4, w, b, dy, "gelu", dt, None, torch.tensor(edges).cuda())
    _check(x, 4, w, b, dy, "gelu", edges, dt, y, dx, dw, db)


@pytest.mark.parametrize("dt,rows,c,groups", [("f32", 60000, 256, 4), ("bf16", 150000, 256, 32), ("f16", 40001, 264, 3)])
def test_samples_beyond_shared_memory(dt, rows, c, groups):
    """One short and one long sample: rows that the CTAs cannot keep are read again."""
    dt = DT[dt]
    edges = [0, 100, rows]
    x, w, b, dy = _data(rows, c, dt, rows)
    y, dx, dw, db = _run(x, groups, w, b, dy, "silu", dt, None, torch.tensor(edges).cuda())
    _check(x, groups, w, b, dy, "silu", edges, dt, y, dx, dw, db)


@pytest.mark.parametrize("dt,n,l,c,groups", [("f32", 3, 300, 4096, 1), ("bf16", 2, 700, 8200, 2), ("f16", 2, 1501, 1030, 2), ("bf16", 700, 33, 1024, 4),
                                             ("f32", 9, 1000, 36, 12), ("bf16", 1, 3, 70000, 7)])
def test_streaming_cuts(dt, n, l, c, groups):
    """Groups wider than one pass of a CTA's threads, odd widths, many samples, in the form of several launches."""
    dt = DT[dt]
    x, w, b, dy = _data(n * l, c, dt, l)
    y, dx, dw, db = _run(x, groups, w, b, dy, "gelu", dt, (n, l, c))
    _check(x, groups, w, b, dy, "gelu", [i * l for i in range(n + 1)], dt, y, dx, dw, db)


@pytest.mark.parametrize("mean", [1e3, -3e4])
def test_large_means(mean):
    x, w, b, dy = _data(4000, 64, torch.float32, 5)
    x += mean
    y, dx, dw, db = _run(x, 8, w, b, dy, "silu", torch.float32, (2, 2000, 64))
    _check(x, 8, w, b, dy, "silu", [0, 2000, 4000], torch.float32, y, dx, dw, db)


def test_strided_rows_and_gradients():
    """The 0e block of [n, 4, 128] features, and an upstream gradient with a stride of its own."""
    g = torch.Generator().manual_seed(1)
    h, up = torch.randn(700, 4, 128, generator=g), torch.randn(700, 3, 128, generator=g)
    w, b = torch.randn(128, generator=g), torch.randn(128, generator=g)
    hd = h.cuda().requires_grad_()
    off = torch.tensor([0, 192, 384, 700]).cuda()
    y = X.group_norm(hd[:, 0], 8, w.cuda(), b.cuda(), activation="silu", offsets=off)
    dh, = torch.autograd.grad(y, hd, up.cuda()[:, 1])
    y0, dx0, _, _ = R.group_norm_grads(h[:, 0], 8, w, b, EPS, "silu", off.tolist(), up[:, 1])
    assert (y.detach().cpu() - y0).abs().max() < 1e-5 and (dh[:, 0].cpu() - dx0).abs().max() < 5e-5 and not dh[:, 1:].any()
    odd = torch.randn(50, 67, generator=g).cuda()[:, 3:]      # rows that start off any vector
    y0 = R.group_norm(odd.cpu().double(), 4, torch.ones(64).double(), torch.zeros(64).double(), EPS, None, [0, 50])
    assert (X.group_norm(odd[None], 4)[0].cpu() - y0).abs().max() < 1e-5


def test_mixed_parameters_and_missing_ones():
    x, w, b, dy = _data(90, 64, torch.bfloat16, 7)
    edges = [0, 30, 60, 90]
    w, b = w.float(), b.float()
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x.view(3, 30, 64), w, b))
    y = X.group_norm(xd, 8, wd, bd, activation="gelu")
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.cuda().view(3, 30, 64))
    assert dw.dtype == db.dtype == torch.float32
    y0, dx0, dw0, db0 = R.group_norm_grads(x, 8, w, b, EPS, "gelu", edges, dy)
    _close(dw, dw0, 1e-3, torch.float32, "dw")                # 90 products of up to 20 each, 2^-17 of them
    _close(db, db0, 1e-3, torch.float32, "db")
    one = torch.ones(64)
    only_b, = torch.autograd.grad(X.group_norm(xd.detach(), 8, None, bd), bd, dy.cuda().view(3, 30, 64))
    _close(only_b, dy.double().sum(0), 1e-4, torch.float32, "db alone")
    only_w, = torch.autograd.grad(X.group_norm(xd.detach(), 8, wd), wd, dy.cuda().view(3, 30, 64))
    _close(only_w, R.group_norm_grads(x, 8, one, 0 * one, EPS, None, edges, dy)[2], 1e-3, torch.float32, "dw alone")
    y = X.group_norm(xd, 8)
    dx, = torch.autograd.grad(y, xd, dy.cuda().view(3, 30, 64))
    y0, dx0, _, _ = R.group_norm_grads(x, 8, one, 0 * one, EPS, None, edges, dy)
    _close(y.reshape(-1, 64), y0, 1e-5, torch.bfloat16, "y")
    _close(dx.reshape(-1, 64), dx0, 1e-5, torch.bfloat16, "dx")


def test_empty_inputs():
    w = torch.ones(16, device="cuda", requires_grad=True)
    for shape, off in (((0, 5, 16), None), ((4, 0, 16), None), ((0, 16), [0]), ((0, 16), [0, 0, 0]), ((6, 16), [2]), ((6, 16), [6, 6])):
        x = torch.randn(*shape, device="cuda", requires_grad=True)
        y = X.group_norm(x, 4, w, offsets=None if off is None else torch.tensor(off).cuda())
        assert y.shape == x.shape and not y.any()
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert not dx.any() and not dw.any()


def test_non_finite_values_stay_in_their_group():
    x = torch.randn(2, 40, 64, device="cuda")
    clean = X.group_norm(x, 8, activation="silu")
    for v in (float("nan"), float("inf"), -float("inf")):
        bad = x.clone()
        bad[1, 3, 17] = v
        y = X.group_norm(bad, 8, activation="silu")
        assert y[1, :, 16:24].isnan().all()
        y[1, :, 16:24] = clean[1, :, 16:24]
        assert torch.equal(y, clean)


def test_bad_offsets_are_nan_and_stay_in_range():
    x = torch.randn(100, 32, device="cuda")
    y = X.group_norm(x, 4, offsets=torch.tensor([-5, 20, 60, 200]).cuda())
    assert y[:20].isnan().all() and y[20:60].isfinite().all() and y[60:].isnan().all()
    y = X.group_norm(x, 4, offsets=torch.tensor([0, 50, 30, 100]).cuda())
    assert y[50:].isnan().all()


def test_refusals():
    x = torch.randn(2, 3, 12, device="cuda")
    with pytest.raises(RuntimeError, match="do not split"):
        X.group_norm(x, 5)
    with pytest.raises(ValueError, match="activation"):
        X.group_norm(x, 4, activation="tanh")
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        X.group_norm(x.double(), 4)
    with pytest.raises(RuntimeError, match="must be"):
        X.group_norm(x[0, 0], 4)
    with pytest.raises(RuntimeError, match="weight / bias must be"):
        X.group_norm(x, 4, torch.ones(11, device="cuda"))
    with pytest.raises(RuntimeError, match="differ in type"):
        X.group_norm(x.half(), 4, torch.ones(12, device="cuda"), torch.ones(12, device="cuda").half())
    with pytest.raises(RuntimeError, match="with offsets"):
        X.group_norm(x, 4, offsets=torch.tensor([0, 2]).cuda())
    with pytest.raises(RuntimeError, match="offsets must be"):
        X.group_norm(x[0], 4, offsets=torch.tensor([0.0, 2.0]).cuda())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        X.group_norm(x[0], 4, offsets=torch.tensor([0, 2]))
    with pytest.raises(RuntimeError, match="eps"):
        X.group_norm(x, 4, eps=-1.0)
    with pytest.raises(RuntimeError, match="once"):
        y = X.group_norm(x.requires_grad_(), 4)
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_gradients_against_differences():
    x, w, b, dy = _data(24, 16, torch.float32, 11)
    y = lambda t: (R.group_norm(t.double(), 4, w.double(), b.double(), EPS, "gelu", [0, 12, 24]) * dy.double()).sum()  # noqa: E731
    xd = x.cuda().requires_grad_()
    out = X.group_norm(xd.view(2, 12, 16), 4, w.cuda(), b.cuda(), activation="gelu")
    dx, = torch.autograd.grad(out, xd, dy.cuda().view(2, 12, 16))
    g, h = torch.Generator().manual_seed(2), 1e-4
    for _ in range(5):
        v = torch.randn(24, 16, generator=g, dtype=torch.float64)
        num = (y(x.double() + h * v) - y(x.double() - h * v)) / (2 * h)
        assert abs(float((dx.cpu().double() * v).sum() - num)) < 1e-4 * float(dx.norm() * v.norm())


def test_streams_and_graphs():
    x, w, b, dy = _data(400, 64, torch.float32, 13)
    xd, wd, bd, dyd = (t.cuda() for t in (x, w, b, dy))
    off = torch.tensor([0, 100, 400]).cuda()

    def step():
        ins = [t.detach().requires_grad_() for t in (xd, wd, bd)]
        y = X.group_norm(ins[0], 8, ins[1], ins[2], activation="silu", offsets=off)
        return (y.detach(), *torch.autograd.grad(y, ins, dyd))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    off.copy_(torch.tensor([0, 250, 400]))                    # lengths may change between replays
    xd.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(step(), held))
