"""A check of group norm's outputs and gradients that sees each term of the formulas (tests only).

Inputs: dy = 1 + xh + noise, so that both means of the backward pass, mean(a) and mean(a xh), are of order one in samples of any length,
and the sums over rows that give dw and db are as large as the sums of their terms' sizes.

Bounds.  u is half a step of the type (and half of its smallest value), e = (8 + log2 M) 2^-23 for groups of M values: x - mean is off by e of the largest |x - mean| and of
|x|, at most 8 standard deviations here, so xh by 8 e.  y (slope at most 1.13) and f' (0.8) follow; dx is r times a sum of four terms
of a size that dy w gives, each off by at most 8 e (1 + |xh|) and f' slopes, together 100 e of the norm of r dy w; dw and db are
off by 20 e of the sums of their terms' sizes |dy| (1 + |xh|) w."""
import math

import torch

import readout_refs as R

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half of the smallest value
EPS = 1e-5


def inputs(rows, c, groups, edges, dt, seed, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=device)

    x = (randn(rows, c) * 2 + 0.5 * randn(c)).to(dt)
    w, b = (1 + 0.3 * randn(c)).to(dt), (0.3 * randn(c)).to(dt)
    one = torch.ones(c, dtype=torch.float64, device=device)
    xh = R.group_norm(x.double(), groups, one, 0 * one, EPS, None, edges)
    return x, w, b, (1 + xh + 0.5 * randn(rows, c)).to(dt)


def failures(x, groups, w, b, dy, act, edges, dt, y, dx, dw, db):
    """What is off: a list of names (empty: all is within the bounds)."""
    y0, dx0, dw0, db0 = R.group_norm_grads(x, groups, w, b, EPS, act, edges, dy)
    one = torch.ones_like(w, dtype=torch.float64)
    xh = R.group_norm(x.double(), groups, one, 0 * one, EPS, None, edges)
    m = max(hi - lo for lo, hi in zip(edges, edges[1:])) * (x.shape[1] // groups)
    u, e = U[dt], (8 + math.log2(m)) * 2.0 ** -23
    wmax, bad = float(w.abs().max()), []
    y, dx, dw, db = (t.detach().double() for t in (y, dx, dw, db))
    if not bool(((y - y0).abs() <= u * y0.abs() + LEAST[dt] + 10 * e * (1 + wmax * (1 + xh.abs()))).all()):
        bad.append("y")

    def by_group(t):                                          # norms of each sample's groups
        return torch.stack([t[lo:hi].reshape(hi - lo, groups, -1).square().sum((0, 2)).sqrt() for lo, hi in zip(edges, edges[1:]) if hi > lo])

    off, want = by_group(dx - dx0), by_group(dx0)
    scale = torch.zeros_like(x, dtype=torch.float64)
    for lo, hi in zip(edges, edges[1:]):
        if hi > lo:
            v = x[lo:hi].double().reshape(hi - lo, groups, -1)
            scale[lo:hi] = (1 / (v.var((0, 2), unbiased=False, keepdim=True) + EPS).sqrt()).expand_as(v).reshape(hi - lo, -1)
    if not bool((off <= u * want + LEAST[dt] * by_group(torch.ones_like(dx0)) + 100 * e * by_group(scale * dy.double() * w.double())).all()):
        bad.append("dx")
    terms = (dy.double().abs() * (1 + xh.abs())).sum(0) * 20 * e * max(1.0, wmax)
    for name, got, ref in (("dw", dw, dw0), ("db", db, db0)):
        tol = u * ref.abs() + LEAST[dt] + terms
        over = (ref.abs() + tol > torch.finfo(dt).max) & (got == ref.sign() * float("inf"))   # beyond float16's 65504
        if bool((~((got - ref).abs() <= tol) & ~over).any()):
            bad.append(name)
    if any(bool(t[:edges[0]].any()) or bool(t[edges[-1]:].any()) for t in (y, dx)):
        bad.append("rows of no sample")
    return bad
