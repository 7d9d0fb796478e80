"""Plain fp64 forms of layer norm, expert routing and expert products (one row / one expert at a time), the checkers of
tests/test_experts.py and tests/test_gpu_experts.py.  The product forms also return the sums of absolute products that
the rounding bounds are stated in."""
import math

import torch


def layer_norm(x, w, b, eps, dy=None):
    x = x.double()
    d = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * r
    w64 = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(d, dtype=torch.float64) if b is None else b.double()
    y = xh * w64 + b64
    if dy is None:
        return y
    dy = dy.double()
    a = dy * w64
    dx = r * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    return y, dx, (dy * xh).reshape(-1, d).sum(0), dy.reshape(-1, d).sum(0)


def _key(v):
    return math.inf if v != v else v


def route(logits, k, bias=None, score="softmax", groups=1, top_groups=1, renormalize=True, scale=1.0):
    """Row by row with Python's sort.  Returns (weights, experts, gap): gap [T] is the smallest difference that decided the
    choice between two values that carry roundings (group values, and biased scores; logits compare exactly)."""
    L = logits.double()
    T, E = L.shape
    W = torch.zeros(T, k, dtype=torch.float64)
    X = torch.full((T, k), -1, dtype=torch.int64)
    gap = torch.full((T,), math.inf, dtype=torch.float64)
    for t in range(T):
        l = L[t].tolist()
        if score == "softmax":
            m = max((v for v in l if v == v), default=0.0)
            m = 0.0 if m == -math.inf else m
            ex = [math.exp(v - m) if v < math.inf else math.nan for v in l]
            tot = sum(ex)
            s = [v / tot if tot != 0 else 0.0 for v in ex]
        else:
            s = [v if v != v else (1 / (1 + math.exp(-v)) if v > -700 else 0.0) for v in l]
        rank = s if bias is None else [s[i] + float(bias[i]) for i in range(E)]
        open_ = [i for i in range(E) if not (l[i] == -math.inf or (bias is not None and rank[i] == -math.inf))]
        if groups > 1:
            per = E // groups
            val = []
            for g in range(groups):
                best = sorted((_key(rank[i]) for i in open_ if i // per == g), reverse=True)[:2]
                if best:
                    val.append((sum(best), g))
            val.sort(key=lambda p: (-p[0], p[1]))
            if len(val) > top_groups:
                gap[t] = min(gap[t], abs(val[top_groups - 1][0] - val[top_groups][0]))
            keep = {g for _, g in val[:top_groups]}
            open_ = [i for i in open_ if i // per in keep]
        key = {i: _key(l[i] if bias is None else rank[i]) for i in open_}
        order = sorted(open_, key=lambda i: (-key[i], i))
        for a, b in zip(order[:k], order[1:k + 1]) if bias is not None else ():
            gap[t] = min(gap[t], abs(key[a] - key[b]))
        sel = order[:k]
        tot = sum(s[i] for i in sel) if renormalize else 1.0
        for j, i in enumerate(sel):
            X[t, j] = i
            W[t, j] = scale * s[i] / tot if tot != 0 else 0.0
    return W, X, gap


def route_weights(logits, experts, score="softmax", renormalize=True, scale=1.0):
    """The weights of a given choice, by torch operations in the type of the logits (for autograd)."""
    s = torch.softmax(logits, 1) if score == "softmax" else torch.sigmoid(logits)
    some = experts >= 0
    sel = torch.where(some, s.gather(1, experts.clamp(min=0)), torch.zeros((), dtype=s.dtype))
    if renormalize:
        tot = sel.sum(1, keepdim=True)
        sel = sel / torch.where(tot == 0, torch.ones_like(tot), tot)
    return scale * sel


def expert_linear(x, w, experts, weights=None, dy=None):
    """out and, with dy, (dx, dw, dweights); every result as a pair (value, sum of the absolute products in it)."""
    T, k = experts.shape
    E, O, D = w.shape
    slots = x.dim() == 3
    x64, w64 = x.double(), w.double()
    Z = torch.zeros(T, k, O, dtype=torch.float64)
    Za = torch.zeros_like(Z)
    g = torch.ones(T, k, dtype=torch.float64) if weights is None else weights.double()
    for t in range(T):
        for j in range(k):
            e = int(experts[t, j])
            if e >= 0:
                xs = x64[t, j] if slots else x64[t]
                Z[t, j] = w64[e] @ xs
                Za[t, j] = w64[e].abs() @ xs.abs()
    if weights is None:
        out, outa = Z, Za
    else:
        out, outa = (g[..., None] * Z).sum(1), (g.abs()[..., None] * Za).sum(1)
    if dy is None:
        return out, outa
    dy = dy.double()
    dx, dw = torch.zeros_like(x64), torch.zeros_like(w64)
    dxa, dwa = torch.zeros_like(dx), torch.zeros_like(dw)
    dg, dga = torch.zeros(T, k, dtype=torch.float64), torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(experts[t, j])
            if e < 0:
                continue
            up = dy[t] if weights is not None else dy[t, j]
            xs = x64[t, j] if slots else x64[t]
            dg[t, j], dga[t, j] = (up * Z[t, j]).sum(), (up.abs() * Za[t, j]).sum()
            dz = g[t, j] * up
            at = (t, j) if slots else (t,)
            dx[at] += w64[e].T @ dz
            dxa[at] += w64[e].abs().T @ dz.abs()
            dw[e] += torch.outer(dz, xs)
            dwa[e] += torch.outer(dz.abs(), xs.abs())
    return (out, outa), (dx, dxa), (dw, dwa), (dg, dga)
