"""Cases of the readout operators: group norm with an activation, products in 8-bit integers, orthogonalised updates.

In plain torch and through the package.  Case keys: "op" (gn, int8, orth), "dtype", and the sizes of the operator.
Sizes are those of the per-atom features: 128 channels per component, feature rows of 4 x 128 per atom, chunks of
16,384 atoms, the 192-atom and 24,000-atom water boxes, 89 elements, 8 experts of 64 hidden channels; the rest are generic.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
# coefficients of the odd polynomial a s + b s^3 + c s^5 that moves every singular value towards one
POLY = (3.4445, -4.7750, 2.0315)
STEPS, ORTH_EPS = 5, 1e-7


def _package():
    root = os.path.join(os.getcwd(), "mace-million_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


# ---------------------------------------------------------------------------------------------------------- cases
def _gn(name, n, length, c, groups, act, dtype, train, ragged=False):
    return {"name": name, "op": "gn", "n": n, "l": length, "c": c, "groups": groups, "act": act, "dtype": dtype,
            "train": train, "ragged": ragged}


def _int8(name, t, k, n, dtype, bias=True):
    return {"name": name, "op": "int8", "t": t, "k": k, "n": n, "dtype": dtype, "bias": bias}


def _orth(name, batch, m, n, dtype):
    return {"name": name, "op": "orth", "batch": batch, "m": m, "n": n, "dtype": dtype}


def listed():
    return [
        # the scalar features of the 192-atom cell as one sample, without gradients: an MD step, latency
        _gn("gn_1x192x128_f32", 1, 192, 128, 8, "silu", "f32", False),
        # a batch of structures of different sizes, one after the other in one tensor
        _gn("gn_train_ragged_384x63x128_f16", 384, 63, 128, 8, "gelu", "f16", True, True),
        # the 24,000-atom box as one sample, all four components' channels
        _gn("gn_train_1x24000x512_f32", 1, 24000, 512, 32, "silu", "f32", True),
        # a large batch of large samples
        _gn("gn_train_64x2048x512_bf16", 64, 2048, 512, 32, "silu", "bf16", True),
        # one token: latency and the bandwidth of the weights
        _int8("int8_1x1024x1024_bf16", 1, 1024, 1024, "bf16", False),
        # the 192-atom cell through the wide linear map
        _int8("int8_192x128x512_f32", 192, 128, 512, "f32"),
        # the 24,000-atom box and one, odd widths
        _int8("int8_24001x515x1001_f16", 24001, 515, 1001, "f16"),
        # a chunk of 16,384 atoms through wide layers
        _int8("int8_16384x4096x4096_bf16", 16384, 4096, 4096, "bf16"),
        # the first matrices of 8 experts: the smallest training step
        _orth("orth_8x64x128_f32", 8, 64, 128, "f32"),
        # one matrix for each element, tall
        _orth("orth_89x512x128_bf16", 89, 512, 128, "bf16"),
        # odd sizes
        _orth("orth_3x515x1023_f16", 3, 515, 1023, "f16"),
        # a large square matrix
        _orth("orth_1x4096x4096_bf16", 1, 4096, 4096, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly multiples of 8 as trained models have them, odd ones among them."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.25 else max(8, w // 8 * 8)


def draw(rng):
    op = rng.choice(["gn", "int8", "orth"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "gn":
        groups = rng.choice([1, 4, 8, 8, 16, 32])
        c = groups * (_width(rng, 4, 64) if rng.random() < 0.25 else 4 * _log(rng, 1, 16))
        n = _log(rng, 1, 1024)
        length = _log(rng, 1, max(1, min(32768, (1 << 26) // (n * c * (2 if dtype == "f32" else 1)))))
        c = _gn("", n, length, c, groups, rng.choice(["none", "silu", "gelu", "relu"]), dtype, rng.random() < 0.6,
                rng.random() < 0.4)
    elif op == "int8":
        k, n = _width(rng, 64, 4096), _width(rng, 64, 4096)
        c = _int8("", _log(rng, 1, 16384), k, n, dtype, rng.random() < 0.5)
    else:
        m, n = _width(rng, 16, 2048), _width(rng, 16, 2048)
        most = int(work(_orth("", 1, 2048, 2048, dtype))["flops"] / work(_orth("", 1, m, n, dtype))["flops"])
        c = _orth("", _log(rng, 1, max(1, min(64, most))), m, n, dtype)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _quantize(x):
    """Rows in 8 bits: scale = largest magnitude / 127 in 32 bits, values the nearest whole multiples of it."""
    top = x.float().abs().amax(-1)
    scale = (top.double() / 127).float()
    q = x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[:, None]
    return torch.where(scale[:, None] > 0, torch.round(q), torch.zeros_like(q)), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "gn":
        n, length, c = case["n"], case["l"], case["c"]
        if case["ragged"]:  # lengths between nothing and twice the mean, the same total for every seed
            cut = torch.rand(n, generator=g, device="cuda") * 2
            at = torch.cumsum(cut, 0)
            at = torch.round(at / at[-1] * (n * length)).long()
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), at]).to(torch.int32)
            shape = (n * length, c)
        else:
            s["offsets"], shape = None, (n, length, c)
        # features of some spread around a mean of their channel
        s["x"] = _randn(g, *shape).mul_(1.5).add_(_randn(g, c)).to(dt)
        s["w"] = (1 + 0.2 * _randn(g, c)).to(dt)
        s["b"] = (0.2 * _randn(g, c)).to(dt)
        if case["train"]:
            s["dy"] = _randn(g, *shape).to(dt)
    elif case["op"] == "int8":
        t, k, n = case["t"], case["k"], case["n"]
        # some channels of the activations are larger than others
        s["x"] = (_randn(g, t, k) * (1 + 2 * torch.rand(k, generator=g, device="cuda"))).to(dt)
        w = torch.empty(n, k, device="cuda").normal_(0.0, k ** -0.5, generator=g)
        q, s["ws"] = _quantize(w)
        # kept as a program keeps them: rows of whole 16 bytes
        s["wq"] = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k].copy_(q)
        s["b"] = (0.2 * _randn(g, n)).to(dt) if case["bias"] else None
    else:
        b, m, n = case["batch"], case["m"], case["n"]
        # momentum: a few strong directions over a floor of noise
        r = max(1, min(m, n) // 8)
        strong = _randn(g, b, m, r) * torch.logspace(0, -2, r, device="cuda") @ _randn(g, b, r, n)
        s["g"] = ((strong + 0.05 * _randn(g, b, m, n)) * 1e-3).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _erf_pdf(z):
    return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)), torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _act(z, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c, p = _erf_pdf(z)
        return z * c, c + z * p
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    return z, torch.ones_like(z)


def _group_mean(v, seg, count, groups, n):
    """Mean of v [rows, C] over the rows and channels of each group of each sample: [rows, C] again."""
    c = v.shape[1]
    if seg is None:
        m = v.view(n, -1, groups, c // groups).mean((1, 3))
        return m.repeat_interleave(c // groups, 1).repeat_interleave(v.shape[0] // n, 0)
    by_channel = torch.zeros(n, c, dtype=v.dtype, device=v.device).index_add_(0, seg, v)
    m = by_channel.view(n, groups, -1).sum(2) / (count[:, None] * (c // groups)).clamp(min=1)
    return m.repeat_interleave(c // groups, 1)[seg]


def _gn_plain(s):
    c, dt = s["case"], s["x"].dtype
    ch, n, groups = c["c"], c["n"], c["groups"]
    x, w, b = s["x"].float().reshape(-1, ch), s["w"].float(), s["b"].float()
    seg = count = None
    if s["offsets"] is not None:
        off = s["offsets"].long()
        count = (off[1:] - off[:-1]).float()
        seg = torch.searchsorted(off[1:], torch.arange(x.shape[0], device=x.device), right=True)
    x = x - _group_mean(x, seg, count, groups, n)
    r = 1 / torch.sqrt(_group_mean(x * x, seg, count, groups, n) + EPS)
    xh = x * r
    y, d = _act(xh * w + b, c["act"])
    out = {"y": y.to(dt).view(s["x"].shape)}
    if not c["train"]:
        return out
    dz = s["dy"].float().reshape(-1, ch) * d
    a = dz * w
    dx = r * (a - _group_mean(a, seg, count, groups, n) - xh * _group_mean(a * xh, seg, count, groups, n))
    return out | {"dx": dx.to(dt).view(s["x"].shape), "dw": (dz * xh).sum(0).to(dt), "db": dz.sum(0).to(dt)}


def _int8_plain(s):
    """Sums of products pass 2^24, so the product of the whole numbers is taken in 64 bits."""
    q, scale = _quantize(s["x"])
    y = (q @ s["wq"].double().T).float() * scale[:, None] * s["ws"]
    return {"y": (y if s["b"] is None else y + s["b"].float()).to(s["x"].dtype)}


def _orth_plain(s):
    a, b, c = POLY
    x = s["g"].float()
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + ORTH_EPS)
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    for _ in range(STEPS):
        p = x @ x.transpose(1, 2)
        x = a * x + (b * p + c * (p @ p)) @ x
    return {"u": (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()}


# ---------------------------------------------------------------------------------------------------------- the package
def _gn_own(s):
    _package()
    from mace_onegpu import readout

    c = s["case"]
    act = None if c["act"] == "none" else c["act"]
    if not c["train"]:
        return {"y": readout.group_norm(s["x"], c["groups"], s["w"], s["b"], eps=EPS, activation=act, offsets=s["offsets"])}
    x, w, b = (s[n].detach().requires_grad_() for n in ("x", "w", "b"))
    y = readout.group_norm(x, c["groups"], w, b, eps=EPS, activation=act, offsets=s["offsets"])
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _int8_own(s):
    _package()
    from mace_onegpu import readout

    return {"y": readout.int8_linear(s["x"], s["wq"], s["ws"], s["b"])}


def _orth_own(s):
    _package()
    from mace_onegpu import optim

    return {"u": optim.orthogonalize(s["g"], steps=STEPS, coefficients=POLY, eps=ORTH_EPS)}


def run(state):
    form = {"gn": (_gn_plain, _gn_own), "int8": (_int8_plain, _int8_own), "orth": (_orth_plain, _orth_own)}
    return form[state["case"]["op"]][1 if own else 0](state)


# ---------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "gn":
        size, e, c = _SIZE[case["dtype"]], case["n"] * case["l"] * case["c"], case["c"]
        train = case["train"]
        # x and y, and dy and dx; the parameters and their gradients
        return {"bytes": size * (e * (4 if train else 2) + c * (4 if train else 2)), "flops": e * (30 if train else 12)}
    if case["op"] == "int8":
        size, t, k, n = _SIZE[case["dtype"]], case["t"], case["k"], case["n"]
        return {"bytes": t * k * size + n * k + 4 * n + (n * size if case["bias"] else 0) + t * n * size,
                "flops": 2 * t * k * n}
    size, b, r, l = _SIZE[case["dtype"]], case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # half of the two symmetric products, the whole of the third
    return {"bytes": b * r * l * (size + 2), "flops": b * STEPS * (r * r * l + r * r * r + 2 * r * r * l)}


# ---------------------------------------------------------------------------------------------------------- 64 bits
def _gn_exact(case, s):
    """Sample by sample: x centred, then its derivatives by the chain rule through mean and variance."""
    c, groups = case["c"], case["groups"]
    per = c // groups
    x = s["x"].double().reshape(-1, c)
    w, b = s["w"].double().view(1, groups, per), s["b"].double().view(1, groups, per)
    if s["offsets"] is None:
        edge = [i * case["l"] for i in range(case["n"] + 1)]
    else:
        edge = s["offsets"].tolist()
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros(c, dtype=torch.float64, device=x.device), torch.zeros(c, dtype=torch.float64, device=x.device)
    for lo, hi in zip(edge, edge[1:]):
        if hi == lo:
            continue
        v = x[lo:hi].view(-1, groups, per)
        var, mean = torch.var_mean(v, dim=(0, 2), unbiased=False, keepdim=True)
        sd = torch.sqrt(var + EPS)
        u = v - mean
        z = torch.addcmul(b, u / sd, w)
        if case["act"] == "silu":
            f, df = z * torch.sigmoid(z), torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))
        elif case["act"] == "gelu":
            cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
            f, df = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        elif case["act"] == "relu":
            f, df = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0)
        else:
            f, df = z, torch.ones_like(z)
        y[lo:hi] = f.reshape(-1, c)
        if case["train"]:
            dz = s["dy"].double().reshape(-1, c)[lo:hi].view_as(v) * df
            dw += (dz * u / sd).sum(0).reshape(-1)
            db += dz.sum(0).reshape(-1)
            dhat = dz * w
            m = v.shape[0] * per
            dvar = -(dhat * u).sum((0, 2), keepdim=True) / (2 * sd ** 3)
            dmean = -dhat.sum((0, 2), keepdim=True) / sd
            dx[lo:hi] = (dhat / sd + 2 * u * dvar / m + dmean / m).reshape(-1, c)
    shape = s["x"].shape
    res = {"y": y.view(shape)}
    return res | {"dx": dx.view(shape), "dw": dw, "db": db} if case["train"] else res


def _int8_exact(case, s):
    x = s["x"].double()
    scale = (x.abs().max(1, keepdim=True).values / 127).float().double()
    q = torch.round(torch.where(scale > 0, x / scale, 0.0))
    y = torch.einsum("tk,nk->tn", q, s["wq"].double()) * (scale * s["ws"].double()[None])
    return {"y": y if s["b"] is None else y + s["b"].double()}


def _orth_exact(case, s):
    """By Horner's rule: x (a + g (b + c g)) with the Gram matrix g of the short side."""
    a, b, c = POLY
    g = s["g"].double()
    x = g / (torch.linalg.vector_norm(g, dim=(1, 2), keepdim=True) + ORTH_EPS)
    for _ in range(STEPS):
        if case["m"] <= case["n"]:
            gram = torch.einsum("bij,bkj->bik", x, x)
            x = torch.baddbmm(x, gram, torch.baddbmm(x, gram, x, beta=b, alpha=c), beta=a)
        else:
            gram = torch.einsum("bji,bjk->bik", x, x)
            x = torch.baddbmm(x, torch.baddbmm(x, x, gram, beta=b, alpha=c), gram, beta=a)
    return {"u": x}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gn": _gn_exact, "int8": _int8_exact, "orth": _orth_exact}[case["op"]](case, s)
