"""The check of group norm's gradients lets the formula through, rounded to the type, and rejects it with any of its terms missing or off by
a part in a hundred: on the CPU, mistakes planted in the oracle."""
import pytest
import torch

import group_norm_checks as C
import readout_refs as R

SHAPES = [([0, 192], 32, 4), ([0, 7000], 16, 2), ([0, 3, 3, 2500, 9001], 24, 3), ([2, 40, 41], 30, 2), ([0, 5], 4096, 1)]


def _by_hand(x, groups, w, b, dy, act, edges, term):
    """y, dx, dw, db from the written formula, with one term changed."""
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    y, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for lo, hi in zip(edges, edges[1:]):
        if hi == lo:
            continue
        v = x[lo:hi].reshape(hi - lo, groups, -1)
        mu, var = v.mean((0, 2), keepdim=True), v.var((0, 2), unbiased=term == "unbiased", keepdim=True)
        r = 1 / (var + C.EPS).sqrt()
        if term == "mean 1% off":
            mu = mu + 0.01 / r
        xh = (v - mu) * r
        z = (xh.reshape(hi - lo, -1) * w + b).requires_grad_()
        f = R.activation(z, act)
        slope, = torch.autograd.grad(f.sum(), z)
        y[lo:hi] = f.detach()
        dz = dy[lo:hi] * (slope if term != "slope of the activation" else 1.0)
        a = (dz * (w if term != "weight in dx" else 1.0)).reshape(hi - lo, groups, -1)
        m1, m2 = a.mean((0, 2), keepdim=True), (a * xh).mean((0, 2), keepdim=True)
        keep = {"mean(a)": (0, 1), "mean(a xh)": (1, 0), "both means": (0, 0), "mean(a) 1% off": (0.99, 1), "mean(a xh) 1% off": (1, 0.99)}
        k1, k2 = keep.get(term, (1, 1))
        dx[lo:hi] = ((r if term != "1 / std" else 1.0) * (a - k1 * m1 - k2 * xh * m2)).reshape(hi - lo, -1)
        dw += (dz * xh.reshape(hi - lo, -1)).sum(0) * (0 if term == "dw" else 0.99 if term == "dw 1% off" else 1)
        db += dz.sum(0) * (0 if term == "db" else 0.99 if term == "db 1% off" else 1)
    if term == "last row":
        dx[edges[-1] - 1] = 0
    if term == "last channel":
        dw[-1] = 0
    return y, dx, dw, db


TERMS = ["mean(a)", "mean(a xh)", "both means", "mean(a) 1% off", "mean(a xh) 1% off", "weight in dx", "slope of the activation", "1 / std", "dw",
         "db", "dw 1% off", "db 1% off", "last channel", "mean 1% off"]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("edges,c,groups", SHAPES)
def test_formula_passes_and_mistakes_do_not(edges, c, groups, dt):
    rows = edges[-1] + 1
    x, w, b, dy = C.inputs(rows, c, groups, edges, dt, c)
    for act in (None, "silu", "gelu"):
        out = [t.to(dt) for t in _by_hand(x, groups, w, b, dy, act, edges, "")]
        assert C.failures(x, groups, w, b, dy, act, edges, dt, *out) == []
        for term in TERMS:
            if (term == "slope of the activation" and act is None) or (dt == torch.bfloat16 and "1%" in term):
                continue                                       # (1% is two steps of bfloat16)
            out = [t.to(dt) for t in _by_hand(x, groups, w, b, dy, act, edges, term)]
            assert C.failures(x, groups, w, b, dy, act, edges, dt, *out), (term, act)
    out = [t.to(dt) for t in _by_hand(x, groups, w, b, dy, None, edges, "")]
    out[0][-1] = 1.0                                           # a row of no sample
    assert C.failures(x, groups, w, b, dy, None, edges, dt, *out)
