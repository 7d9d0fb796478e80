"""Cases of the expert-routing operators: layer norm, routing and expert products, in plain torch and through the package.

Case keys: "op" (ln, route, expert), "train" (the backward pass too), "dtype", and the sizes of the operator.
Sizes are those of the per-atom features: 128 channels per component, feature rows of 4 x 128 per atom,
chunks of 16,384 atoms, the 192-atom and 24,000-atom water boxes, 89 elements; the rest are generic.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def _ops():
    """The package's public module."""
    root = os.path.join(os.getcwd(), "mace-million_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mace_onegpu import experts

    return experts


# ---------------------------------------------------------------------------------------------------------- cases
def _ln(name, n, d, dtype, train, stride=0):
    return {"name": name, "op": "ln", "train": train, "dtype": dtype, "n": n, "d": d, "stride": stride or d}


def _route(name, t, e, k, dtype, score, train, groups=1, top_groups=1, bias=False, renorm=True, masked=False):
    return {"name": name, "op": "route", "train": train, "dtype": dtype, "t": t, "e": e, "k": k, "score": score,
            "groups": groups, "top_groups": top_groups, "bias": bias, "renorm": renorm, "masked": masked}


def _expert(name, t, e, k, d, o, dtype, train, combine=True, masked=False):
    return {"name": name, "op": "expert", "train": train, "dtype": dtype, "t": t, "e": e, "k": k, "d": d, "o": o,
            "combine": combine, "masked": masked}


def listed():
    return [
        # the scalar (0e) block of the features of the 192-atom cell, rows 4 x 128 apart: an MD step, latency
        _ln("ln_192x128_f32", 192, 128, "f32", False, 512),
        # the same block of one chunk of 16,384 atoms in a training step
        _ln("ln_train_16384x128_f32", 16384, 128, "f32", True, 512),
        # odd width and row count
        _ln("ln_train_24001x515_bf16", 24001, 515, "bf16", True),
        # wide features of a large batch
        _ln("ln_train_65536x2048_bf16", 65536, 2048, "bf16", True),
        # one token, grouped sigmoid scores with a balance bias: latency
        _route("route_1x64_f32", 1, 64, 4, "f32", "sigmoid", False, 8, 4, True),
        # two experts of as many as there are elements for the 24,000-atom box, some experts closed to some atoms
        _route("route_train_24000x89_f32", 24000, 89, 2, "f32", "softmax", True, renorm=False, masked=True),
        # a large batch of the grouped router
        _route("route_train_131072x128_bf16", 131072, 128, 8, "bf16", "sigmoid", True, 8, 4, True),
        # one token through 4 of 64 experts: latency and the bandwidth of the weights
        _expert("expert_1_e64_1024_bf16", 1, 64, 4, 1024, 1024, "bf16", False),
        # the 192-atom cell through fp32 experts over 128 channels
        _expert("expert_192_e8_128_f32", 192, 8, 2, 128, 128, "f32", False),
        # a chunk of atoms, one linear map out of 89 for each, fp32, per-slot outputs, some atoms without an expert
        _expert("expert_train_16384_e89_f32", 16384, 89, 1, 128, 512, "f32", True, combine=False, masked=True),
        # the 24,000-atom box, odd output width
        _expert("expert_train_24000_e16_f16", 24000, 16, 2, 512, 515, "f16", True),
        # a large training batch
        _expert("expert_train_65536_e64_bf16", 65536, 64, 4, 1024, 2048, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly multiples of 8 as trained models have them, odd ones among them."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.25 else max(8, w // 8 * 8)


def draw(rng):
    op = rng.choice(["ln", "route", "expert", "expert"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    if op == "ln":
        d = _width(rng, 64, 4096)
        n = _log(rng, 1, min(131072, 65536 * 2048 // d))
        c = _ln("", n, d, dtype, train, d * rng.choice([1, 1, 4]) if n * d < 1 << 25 else d)
    elif op == "route":
        # the bias goes with sigmoid scores, whose value for an expert does not hang on the sum over the others
        groups = rng.choice([1, 1, 4, 8])
        per = rng.randint(1 if groups == 1 else 2, 256 // groups)
        e = groups * per
        top = rng.randint(1, groups)
        score = rng.choice(["softmax", "sigmoid"])
        c = _route("", _log(rng, 1, 131072), e, rng.randint(1, min(8, top * per)), dtype, score, train, groups, top,
                   score == "sigmoid" and rng.random() < 0.7, rng.random() < 0.6, rng.random() < 0.3)
    else:
        e, d, o = _log(rng, 2, 128), _width(rng, 64, 2048), _width(rng, 64, 2048)
        k = rng.randint(1, min(8, e))
        t = _log(rng, 1, min(65536, 262144 // k))
        combine = rng.random() < 0.7
        c = _expert("", t, e, k, d, o, dtype, train, combine, rng.random() < 0.3)
        while work(c)["flops"] > 1.5e12 or t * k * o * (1 if combine else 2) > 1 << 28:
            t = max(1, t // 2)
            c["t"] = t
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "ln":
        n, d = case["n"], case["d"]
        # features of some spread around a mean of their own, as trained ones have
        rows = _randn(g, n, case["stride"]).mul_(1.5).add_(_randn(g, n, 1)).to(dt)
        s["x"] = rows[:, :d]
        s["w"] = (1 + 0.2 * _randn(g, d)).to(dt)
        s["b"] = (0.2 * _randn(g, d)).to(dt)
        if case["train"]:
            s["dy"] = _randn(g, n, d).to(dt)
    elif case["op"] == "route":
        t, e = case["t"], case["e"]
        logits = (_randn(g, t, e) * 1.5 + 0.5 * _randn(g, e)).to(dt)
        if case["masked"]:  # experts closed to a token; some tokens have none
            logits = logits.masked_fill(torch.rand(t, e, generator=g, device="cuda") < 0.3, float("-inf"))
            logits = logits.masked_fill(torch.rand(t, 1, generator=g, device="cuda") < 0.02, float("-inf"))
        s["logits"] = logits
        s["bias"] = 0.1 * _randn(g, e) if case["bias"] else None
        if case["train"]:
            s["dw"] = _randn(g, t, case["k"])
    else:
        t, e, k, d, o = (case[x] for x in ("t", "e", "k", "d", "o"))
        s["x"] = _randn(g, t, d).to(dt)
        s["w"] = torch.empty(e, o, d, dtype=dt, device="cuda").normal_(0.0, d ** -0.5, generator=g)
        # experts of uneven popularity
        l = _randn(g, t, e) + 0.5 * _randn(g, e)
        top = torch.topk(l, k, dim=1)
        experts, p = top.indices, torch.softmax(top.values, 1)
        if case["masked"]:  # atoms without an expert (padding, ghosts)
            experts = experts.masked_fill(torch.rand(t, 1, generator=g, device="cuda") < 0.1, -1)
        s["experts"] = experts.to(torch.int32)
        s["weights"] = p.contiguous() if case["combine"] else None
        if case["train"]:
            s["dy"] = _randn(g, t, o).to(dt) if case["combine"] else _randn(g, t, k, o).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _ln_plain(s):
    c, dt = s["case"], s["x"].dtype
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    x = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    xh = x * r
    y = (xh * w + b).to(dt)
    if not c["train"]:
        return {"y": y}
    dy = s["dy"].float()
    a = dy * w
    dx = r * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dw": (dy * xh).sum(0).to(dt), "db": dy.sum(0).to(dt)}


def _route_plain(s):
    c, l = s["case"], s["logits"].float()
    t, e = l.shape
    k, low = c["k"], float("-inf")
    if c["score"] == "softmax":
        top = l.max(1, keepdim=True).values
        ex = torch.exp(l - torch.where(top == low, torch.zeros_like(top), top))
        total = ex.sum(1, keepdim=True)
        score = torch.where(total > 0, ex / total, ex)
        rank = ex  # in the order of the scores, whatever the sum
    else:
        rank = score = 1 / (1 + torch.exp(-l))
    if s["bias"] is not None:
        rank = score + s["bias"]
    closed = l == low
    key = rank if s["bias"] is not None else l
    if c["groups"] > 1:
        n = c["groups"]
        best = torch.sort(rank.masked_fill(closed, low).view(t, n, -1), dim=2, descending=True).values[:, :, :2]
        value = torch.where(best == low, torch.zeros_like(best), best).sum(2).masked_fill(best[:, :, 0] == low, low)
        chosen = torch.sort(value, dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        keep = torch.zeros(t, n, dtype=torch.bool, device=l.device).scatter_(1, chosen, True)
        closed = closed | ~keep.repeat_interleave(e // n, dim=1)
    got = torch.sort(key.masked_fill(closed, low), dim=1, descending=True, stable=True)
    idx, some = got.indices[:, :k], got.values[:, :k] != low
    sel = torch.where(some, score.gather(1, idx), torch.zeros((), device=l.device))
    if c["renorm"]:
        tot = sel.sum(1, keepdim=True)
        div = torch.where(tot > 0, tot, torch.ones_like(tot))
    else:
        div = torch.ones(t, 1, device=l.device)
    wts = sel / div
    out = {"weights": wts, "experts": torch.where(some, idx, -torch.ones_like(idx)).to(torch.int32)}
    if not c["train"]:
        return out
    ds = s["dw"]
    if c["renorm"]:
        ds = torch.where(tot > 0, (ds - (ds * wts).sum(1, keepdim=True)) / div, torch.zeros_like(ds))
    ds = torch.where(some, ds, torch.zeros_like(ds))
    if c["score"] == "softmax":
        full = torch.zeros_like(l).scatter_(1, idx, ds)
        dl = score * (full - (sel * ds).sum(1, keepdim=True))
    else:
        dl = torch.zeros_like(l).scatter_(1, idx, ds * sel * (1 - sel))
    return out | {"dlogits": dl.to(s["logits"].dtype)}


def _expert_plain(s):
    """Few slots: each slot's matrix is gathered. Else the slots are sorted into one padded batch over the experts."""
    c, dt = s["case"], s["x"].dtype
    t, e, k, d, o = (c[x] for x in ("t", "e", "k", "d", "o"))
    flat = s["experts"].reshape(-1).long()
    token = torch.arange(t * k, device=flat.device) // k
    slot = torch.nonzero(flat >= 0)[:, 0]
    ex, tok = flat[slot], token[slot]
    g = s["weights"].reshape(-1)[slot] if c["combine"] else None
    xs = s["x"].float()[tok]
    few = t * k < e and not c["train"]
    if few:
        z = torch.bmm(s["w"][ex].float(), xs[:, :, None])[:, :, 0]
    else:
        one = torch.zeros(e, slot.numel(), device=flat.device).scatter_(0, ex[None], 1.0)
        count = one.sum(1).long()
        order = torch.sort(ex, stable=True).indices
        start = torch.cumsum(count, 0) - count
        at = torch.empty_like(ex)
        at[order] = torch.arange(ex.numel(), device=ex.device) - start[ex[order]]
        del one
        cap = int(count.max())
        w = s["w"].float()
        xb = torch.zeros(e, cap, d, device=flat.device)
        xb[ex, at] = xs
        z = torch.bmm(xb, w.transpose(1, 2))[ex, at]
    if c["combine"]:
        out = torch.zeros(t, o, device=flat.device).index_add_(0, tok, z * g[:, None])
    else:
        out = torch.zeros(t * k, o, device=flat.device).index_copy_(0, slot, z).view(t, k, o)
    res = {"out": out.to(dt)}
    if not c["train"]:
        return res
    dy = s["dy"].float()
    up = dy[tok] if c["combine"] else dy.view(t * k, o)[slot]
    if c["combine"]:
        dg = torch.zeros(t * k, device=flat.device).index_copy_(0, slot, (up * z).sum(1))
        res["dweights"] = dg.view(t, k)
        up = up * g[:, None]
    del z
    db = torch.zeros(e, cap, o, device=flat.device)
    db[ex, at] = up
    del up
    res["dw"] = torch.bmm(db.transpose(1, 2), xb).to(dt)
    del xb
    dxs = torch.bmm(db, w)[ex, at]
    res["dx"] = torch.zeros(t, d, device=flat.device).index_add_(0, tok, dxs).to(dt)
    return res


# ---------------------------------------------------------------------------------------------------------- the package
def _ln_own(s):
    X = _ops()
    if not s["case"]["train"]:
        return {"y": X.layer_norm(s["x"], s["w"], s["b"], EPS)}
    x, w, b = (s[n].detach().requires_grad_() for n in ("x", "w", "b"))
    y = X.layer_norm(x, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _route_own(s):
    X, c = _ops(), s["case"]
    l = s["logits"].detach().requires_grad_() if c["train"] else s["logits"]
    w, experts = X.route(l, c["k"], bias=s["bias"], score=c["score"], groups=c["groups"], top_groups=c["top_groups"],
                         renormalize=c["renorm"])
    out = {"weights": w.detach(), "experts": experts}
    return out | {"dlogits": torch.autograd.grad(w, l, s["dw"])[0]} if c["train"] else out


def _expert_own(s):
    X, c = _ops(), s["case"]
    plan = X.plan_experts(s["experts"], c["e"])
    if not c["train"]:
        return {"out": X.expert_linear(s["x"], s["w"], plan, s["weights"])}
    x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
    if c["combine"]:
        g = s["weights"].detach().requires_grad_()
        out = X.expert_linear(x, w, plan, g)
        dx, dw, dg = torch.autograd.grad(out, (x, w, g), s["dy"])
        return {"out": out.detach(), "dweights": dg, "dw": dw, "dx": dx}
    out = X.expert_linear(x, w, plan)
    dx, dw = torch.autograd.grad(out, (x, w), s["dy"])
    return {"out": out.detach(), "dw": dw, "dx": dx}


def run(state):
    form = {"ln": (_ln_plain, _ln_own), "route": (_route_plain, _route_own), "expert": (_expert_plain, _expert_own)}
    return form[state["case"]["op"]][1 if own else 0](state)


# ---------------------------------------------------------------------------------------------------------- work
def work(case):
    b = _SIZE[case["dtype"]]
    if case["op"] == "ln":
        n, d = case["n"], case["d"]
        # x and y, and dy and dx; the parameters and their gradients
        return {"bytes": b * (n * d * (4 if case["train"] else 2) + d * (4 if case["train"] else 2)),
                "flops": n * d * (20 if case["train"] else 8)}
    if case["op"] == "route":
        t, e, k = case["t"], case["e"], case["k"]
        return {"bytes": t * (e * b * (2 if case["train"] else 1) + 8 * k + (4 * k if case["train"] else 0)),
                "flops": t * e * (15 if case["train"] else 8)}
    t, e, k, d, o = (case[x] for x in ("t", "e", "k", "d", "o"))
    used = min(e, t * k)
    rows = t if case["combine"] else t * k
    got = t * d * b + used * o * d * b + rows * o * b + 4 * t * k * (2 if case["combine"] else 1)
    if case["train"]:
        got += rows * o * b + t * d * b + e * o * d * b + (4 * t * k if case["combine"] else 0)
    return {"bytes": got, "flops": 2 * t * k * d * o * (3 if case["train"] else 1)}


# ---------------------------------------------------------------------------------------------------------- 64 bits
def _ln_exact(case, s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + EPS)
    hat = (x - mean) / sd
    res = {"y": torch.addcmul(b, hat, w)}
    if case["train"]:
        dy, n = s["dy"].double(), case["d"]
        up = dy * w
        # the Jacobian of (x - mean) / sd applied from the left
        proj = up - up.sum(1, keepdim=True) / n - hat * torch.einsum("td,td->t", up, hat)[:, None] / n
        res |= {"dx": proj / sd, "dw": torch.einsum("td,td->d", dy, hat), "db": torch.einsum("td->d", dy)}
    return res


def _route_exact(case, s):
    """The choice is made from the 64-bit scores by taking the best that is left, k times."""
    l = s["logits"].double()
    t, e = l.shape
    score = torch.softmax(l, 1).nan_to_num(0.0) if case["score"] == "softmax" else torch.sigmoid(l)
    open_ = torch.isfinite(l)
    rank = score if s["bias"] is None else score + s["bias"].double()
    if case["groups"] > 1:
        n = case["groups"]
        by = torch.where(open_, rank, torch.full_like(rank, -1e9)).view(t, n, e // n)
        first, at = by.max(2)
        second = by.scatter(2, at[:, :, None], -1e9).max(2).values
        value = torch.where(second > -1e8, first + second, first)
        for_group = torch.zeros(t, n, dtype=torch.bool, device=l.device)
        for _ in range(case["top_groups"]):
            g = torch.where(for_group, -math.inf, value).max(1).indices
            for_group[torch.arange(t, device=l.device), g] = True
        open_ = open_ & for_group[:, :, None].expand(t, n, e // n).reshape(t, e)
    key = (l if s["bias"] is None else rank).masked_fill(~open_, -math.inf)
    pick = []
    for _ in range(case["k"]):
        v, i = key.max(1)
        pick.append(torch.where(v == -math.inf, -1, i))
        key = key.scatter(1, i[:, None], -math.inf)
    idx = torch.stack(pick, 1)
    hot = torch.zeros(t, case["k"], e, dtype=torch.float64, device=l.device) if t * case["k"] * e < 1 << 28 else None
    some = (idx >= 0).double()
    at = idx.clamp(min=0)
    sel = score.gather(1, at) * some
    tot = sel.sum(1, keepdim=True) if case["renorm"] else torch.ones(t, 1, dtype=torch.float64, device=l.device)
    wts = torch.where(tot > 0, sel / tot, 0.0)
    res = {"weights": wts, "experts": None}
    if case["train"]:
        dw = s["dw"].double() * some
        ds = torch.where(tot > 0, (dw - (dw * wts).sum(1, keepdim=True)) / tot * some, 0.0) if case["renorm"] else dw
        if hot is not None:
            full = torch.einsum("tke,tk->te", hot.scatter_(2, at[:, :, None], 1.0), ds)
        else:
            full = torch.zeros_like(l).scatter_add_(1, at, ds)
        if case["score"] == "softmax":
            res["dlogits"] = score * full - score * (score * full).sum(1, keepdim=True)
        else:
            res["dlogits"] = full * score * (1 - score)
    return res


def _expert_exact(case, s):
    """One expert after the other."""
    t, e, k, d, o = (case[n] for n in ("t", "e", "k", "d", "o"))
    dev, f64 = s["x"].device, torch.float64
    out = torch.zeros((t, o) if case["combine"] else (t, k, o), dtype=f64, device=dev)
    dx, dw = torch.zeros(t, d, dtype=f64, device=dev), torch.zeros(e, o, d, dtype=f64, device=dev)
    dg = torch.zeros(t, k, dtype=f64, device=dev)
    for i in torch.unique(s["experts"]).tolist():
        if i < 0:
            continue
        tok, j = torch.nonzero(s["experts"] == i, as_tuple=True)
        xi, wi = s["x"][tok].double(), s["w"][i].double()
        z = xi @ wi.T
        g = s["weights"][tok, j].double()[:, None] if case["combine"] else None
        if case["combine"]:
            out.index_add_(0, tok, g * z)
        else:
            out[tok, j] = z
        if case["train"]:
            dy = s["dy"][tok].double() if case["combine"] else s["dy"][tok, j].double()
            if case["combine"]:
                dg[tok, j] = (dy * z).sum(1)
                dy = dy * g
            dw[i] = dy.T @ xi
            dx.index_add_(0, tok, dy @ wi)
    res = {"out": out}
    if case["train"]:
        res |= {"dw": dw, "dx": dx} | ({"dweights": dg} if case["combine"] else {})
    return res


def exact(case, seed):
    s = prepare(case, seed)
    return {"ln": _ln_exact, "route": _route_exact, "expert": _expert_exact}[case["op"]](case, s)
