"""Layer norm, expert routing and expert products (mace_onegpu.experts) against the plain fp64 forms of
tests/expert_refs.py: types, strides, odd widths, empty and single rows, closed experts, non-finite values, refusals,
streams, and gradients against the formula's and against differences.

Tolerances.  u(type) is the largest relative error of one rounding to the type: 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32).
A layer norm output is rounded once from fp32 arithmetic over d terms: u |value| plus (8 + log2 d) 2^-23 of the largest
magnitude (pairwise sums).  A product is a sum of K terms in fp32: (8 + K / 8) 2^-23 times the sum of the absolute
products; rows that are summed over k choices and the products' scaled operands are rounded once more: another u of that
sum."""
import math

import pytest
import torch

import expert_refs as R
from mace_onegpu import _native as N
from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E32 = 2.0 ** -23


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cuda(t, grad=False):
    return None if t is None else t.cuda().requires_grad_(grad)


# ------------------------------------------------------------------------------------------------ layer norm
def _ln_close(got, want, d, dt, terms=1):
    want = want.double()
    tol = U[dt] * want.abs() + (8 + math.log2(d * terms + 1)) * E32 * want.abs().max().clamp(min=1.0)
    assert got.dtype == dt and got.shape == want.shape
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(got.double().cpu() - want).abs().max()}"


LN_WIDTHS = [1, 3, 8, 31, 64, 128, 129, 256, 515, 1000, 1024, 2048, 2049, 4096, 5000, 8192, 16384, 16392, 20001]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", LN_WIDTHS)
def test_layer_norm_forward_and_backward(d, dt):
    dt = DT[dt]
    n = 37 if d <= 2048 else 5
    g = _gen(d)
    x = (torch.randn(n, d, generator=g) * 2 + 0.5).to(dt)
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(dt)
    b = (0.3 * torch.randn(d, generator=g)).to(dt)
    dy = torch.randn(n, d, generator=g).to(dt)
    xd, wd, bd = _cuda(x, True), _cuda(w, True), _cuda(b, True)
    y = X.layer_norm(xd, wd, bd)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.cuda())
    y0, dx0, dw0, db0 = R.layer_norm(x, w, b, 1e-5, dy)
    if d == 1:                                    # x - mean = 0: the output is the bias, dx is zero
        assert torch.equal(y.cpu().detach(), b.expand(n, 1)) and not dx.any() and not dw.any()
        return
    _ln_close(y.detach(), y0, d, dt)
    # dx carries 1 / std (up to a few for the narrowest rows) and the sums of d terms
    _ln_close(dx, dx0, d, dt, 8)
    _ln_close(dw, dw0, n, dt, 8)
    _ln_close(db, db0, n, dt, 8)
    assert torch.equal(y.detach(), X.layer_norm(xd.detach(), wd.detach(), bd.detach()))
    again = torch.autograd.grad(X.layer_norm(xd, wd, bd), (xd, wd, bd), dy.cuda())
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))     # fixed order of the sums


@pytest.mark.parametrize("n", [0, 1, 2, 9, 1000, 40001])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layer_norm_rows_and_strides(n, dt):
    """The 0e block of [n, 4, 128] features: rows 512 apart; upstream gradients with a stride of their own."""
    dt = DT[dt]
    g = _gen(n)
    h = torch.randn(n, 4, 128, generator=g).to(dt)
    w = (1 + 0.3 * torch.randn(128, generator=g)).to(dt)
    b = torch.randn(128, generator=g).to(dt)
    up = torch.randn(n, 3, 128, generator=g).to(dt)
    hd, wd, bd = _cuda(h, True), _cuda(w, True), _cuda(b, True)
    y = X.layer_norm(hd[:, 0], wd, bd)
    dh, dw, db = torch.autograd.grad(y, (hd, wd, bd), up.cuda()[:, 1])
    if n == 0:
        assert y.shape == (0, 128) and not dw.any() and not db.any()
        return
    y0, dx0, dw0, db0 = R.layer_norm(h[:, 0], w, b, 1e-5, up[:, 1])
    _ln_close(y.detach(), y0, 128, dt)
    _ln_close(dh[:, 0], dx0, 128, dt, 8)
    assert not dh[:, 1:].any()
    _ln_close(dw, dw0, n, dt, 8)
    _ln_close(db, db0, n, dt, 8)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [4, 24, 40, 72, 136, 520])
def test_layer_norm_narrow_rows_of_many_tokens(d, dt):
    """Several rows to a warp, and more rows than one pass of the grid."""
    dt, n = DT[dt], 100003
    g = _gen(d)
    x = (torch.randn(n, d, generator=g) * 2 - 1).to(dt)
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(dt)
    b = torch.randn(d, generator=g).to(dt)
    dy = torch.randn(n, d, generator=g).to(dt)
    xd, wd, bd = _cuda(x, True), _cuda(w, True), _cuda(b, True)
    y = X.layer_norm(xd, wd, bd)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.cuda())
    y0, dx0, dw0, db0 = R.layer_norm(x, w, b, 1e-5, dy)
    # a few values can have a small deviation 1 / r: x - mean is then off by (log2 d) ulp of the largest |x|, times r
    x, w, b, dy = x.double(), w.double(), b.double(), dy.double()
    c = x - x.mean(1, keepdim=True)
    r = 1 / (c.square().mean(1, keepdim=True) + 1e-5).sqrt()
    off = (8 + math.log2(d)) * E32 * (1 + r * x.abs().amax(1, keepdim=True))
    xh, up = (c * r).abs().amax(1, keepdim=True), (dy * w).abs().amax(1, keepdim=True)
    for got, want, scale in ((y, y0, xh * w.abs().max() + b.abs().max()), (dx, dx0, 8 * r * up * (1 + xh * xh))):
        assert got.dtype == dt and got.shape == want.shape
        assert not ((got.detach().cpu().double() - want).abs() > U[dt] * want.abs() + off * scale).any()
    _ln_close(dw, dw0, n, dt, 8)
    _ln_close(db, db0, n, dt, 8)


def test_layer_norm_views_parameters_and_shapes():
    g = _gen(3)
    base = torch.randn(6, 5, 80, generator=g)
    w32, b32 = torch.rand(64, generator=g) + 0.5, torch.randn(64, generator=g)
    for dt in (torch.float32, torch.bfloat16):
        x = base.to(dt).cuda()
        odd = x[:, :, 3:67]                       # a start that no vector access is aligned to
        want = R.layer_norm(odd.cpu(), w32, b32, 1e-5)
        _ln_close(X.layer_norm(odd, w32.cuda(), b32.cuda()), want, 64, dt)        # fp32 parameters
        _ln_close(X.layer_norm(odd, None, b32.cuda()), R.layer_norm(odd.cpu(), None, b32, 1e-5), 64, dt)
        _ln_close(X.layer_norm(odd, w32.cuda()), R.layer_norm(odd.cpu(), w32, None, 1e-5), 64, dt)
        _ln_close(X.layer_norm(odd), R.layer_norm(odd.cpu(), None, None, 1e-5), 64, dt)
        t = x.transpose(1, 2)                     # last dimension strided: copied
        _ln_close(X.layer_norm(t), R.layer_norm(t.cpu(), None, None, 1e-5), 5, dt, 64)
        one = x[0, 0]
        _ln_close(X.layer_norm(one), R.layer_norm(one.cpu(), None, None, 1e-5), 80, dt)
        xg = odd.detach().requires_grad_()
        wg = w32.cuda().requires_grad_()
        dx, dw = torch.autograd.grad(X.layer_norm(xg, wg).float().sum(), (xg, wg))
        _, dx0, dw0, _ = R.layer_norm(odd.cpu(), w32, None, 1e-5, torch.ones(6, 5, 64))
        assert dw.dtype == torch.float32
        _ln_close(dx, dx0, 64, dt, 8)
        _ln_close(dw, dw0, 30, torch.float32, 8)


def test_layer_norm_non_finite_rows_stay_in_their_rows():
    g = _gen(4)
    x = torch.randn(40, 96, generator=g)
    x[3, 5], x[7, 0], x[11, 95] = float("nan"), float("inf"), -float("inf")
    y = X.layer_norm(x.cuda()).cpu()
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 7, 11]] = True
    assert torch.isnan(y[bad]).any(1).all() and torch.isfinite(y[~bad]).all()
    _ln_close(y[~bad], R.layer_norm(x[~bad], None, None, 1e-5), 96, torch.float32)
    big = torch.full((2, 64), 6e4).half()
    big[1, ::2] = -6e4
    _ln_close(X.layer_norm(big.cuda()), R.layer_norm(big, None, None, 1e-5), 64, torch.float16)


def test_layer_norm_gradient_against_differences():
    """Central differences of the fp64 form along random directions of every input."""
    g = _gen(5)
    x, w, b, dy = (torch.randn(*s, generator=g) for s in ((9, 70), (70,), (70,), (9, 70)))
    xd, wd, bd = _cuda(x, True), _cuda(w, True), _cuda(b, True)
    grads = torch.autograd.grad(X.layer_norm(xd, wd, bd), (xd, wd, bd), dy.cuda())
    h = 1e-5
    for i, gr in enumerate(grads):
        v = torch.randn(gr.shape, generator=g, dtype=torch.float64)
        args = [x.double(), w.double(), b.double()]
        f = [(R.layer_norm(*[a + s * h * v if q == i else a for q, a in enumerate(args)], 1e-5) * dy.double()).sum()
             for s in (1, -1)]
        fd = float((f[0] - f[1]) / (2 * h))
        # differences are exact to h^2 and 1e-16 / h; the kernel's gradient to fp32
        assert abs(float((gr.double().cpu() * v).sum()) - fd) <= 2e-5 * (1 + abs(fd))


def test_layer_norm_refusals():
    x = torch.randn(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    for bad, msg in [(lambda: X.layer_norm(x.double()), "float32, bfloat16 or float16"),
                     (lambda: X.layer_norm(x, w[:8]), "must be \\[16\\]"),
                     (lambda: X.layer_norm(x, w.bfloat16()), "type of x or float32"),
                     (lambda: X.layer_norm(x.bfloat16(), w, w.bfloat16()), "differ in type"),
                     (lambda: X.layer_norm(x, w.cpu()), "CUDA tensor"),
                     (lambda: X.layer_norm(x[:, :0]), "at least 1"),
                     (lambda: X.layer_norm(x, eps=-1.0), "negative")]:
        with pytest.raises(RuntimeError, match=msg):
            bad()
    xg = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(X.layer_norm(xg).pow(2).sum(), xg, create_graph=True)


# ------------------------------------------------------------------------------------------------ routing
ROUTES = [  # E, k, score, groups, top_groups, bias, renormalize, scale
    (1, 1, "softmax", 1, 1, False, True, 1.0),
    (2, 1, "sigmoid", 1, 1, False, False, 1.0),
    (8, 2, "softmax", 1, 1, False, True, 1.0),
    (8, 8, "sigmoid", 2, 1, True, True, 2.5),
    (31, 5, "softmax", 1, 1, True, False, 1.0),
    (64, 6, "sigmoid", 8, 4, True, True, 1.0),
    (89, 2, "softmax", 1, 1, False, False, 1.0),
    (128, 8, "softmax", 8, 3, False, True, 1.0),
    (200, 32, "sigmoid", 4, 2, False, False, 0.5),
    (512, 16, "softmax", 32, 5, True, True, 1.0),
    (512, 3, "sigmoid", 1, 1, True, True, 1.0),
    (50, 4, "sigmoid", 5, 2, False, True, 1.0),
    (510, 7, "softmax", 17, 6, False, False, 1.0),
    (510, 9, "sigmoid", 3, 2, True, True, 1.0),
    (148, 3, "softmax", 4, 2, False, True, 1.0),
    (96, 6, "sigmoid", 32, 9, True, False, 1.0),
]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E,k,score,groups,top,bias,renorm,scale", ROUTES)
def test_route_choice_weights_and_gradient(E, k, score, groups, top, bias, renorm, scale, dt):
    g = _gen(E + k)
    T = 67
    l = (torch.randn(T, E, generator=g) * 2).to(DT[dt])
    if E > 2:
        l = l.masked_fill(torch.rand(T, E, generator=g) < 0.2, float("-inf"))
        l[5] = float("-inf")                      # a row with nothing open
        l[6, 1:] = float("-inf")                  # one open
        l[7] = 0.25                               # all tied
        l[8] = torch.finfo(DT[dt]).min            # the type's lowest value is a logit like any other
    b = 0.3 * torch.randn(E, generator=g) if bias else None
    ld = _cuda(l, True)
    kw = dict(score=score, groups=groups, top_groups=top, renormalize=renorm, scale=scale)
    w, e = X.route(ld, k, bias=_cuda(b), **kw)
    w0, e0, gap = R.route(l, k, b, **kw)
    # the choice is decided in fp32: rows decided by less than a few roundings of the scores are left out
    clear = gap > 1e-6
    clear[7] = True                               # equal scores: the lowest index on both sides
    assert clear.double().mean() > 0.8
    assert torch.equal(e.cpu().long()[clear], e0[clear])
    assert (w.detach().double().cpu() - w0)[clear].abs().max() <= 2e-6 * scale
    assert e.dtype == torch.int32 and w.dtype == torch.float32
    dw = torch.randn(T, k, generator=g)
    dl, = torch.autograd.grad(w, ld, dw.cuda())
    l64 = l.double().requires_grad_()
    safe = l64.masked_fill(torch.isinf(l64).all(1, keepdim=True), 0.0)
    dead = torch.isinf(l).all(1)
    ref = R.route_weights(safe, e.cpu().long(), score, renorm, scale)
    dl0, = torch.autograd.grad(ref, l64, dw.double())
    assert not dl[dead.cuda()].any()
    err = (dl.double().cpu() - dl0).abs()[~dead]
    assert (err <= U[DT[dt]] * dl0.abs()[~dead] + 2e-6 * scale * dw.abs().max()).all()


@pytest.mark.parametrize("E,groups,top", [(64, 8, 4), (200, 4, 2), (200, 8, 3), (148, 4, 2), (89, 1, 1), (510, 17, 5), (12, 1, 1)])
def test_route_many_tokens_agree_with_few(E, groups, top):
    """Many tokens take few lanes each, few tokens a whole warp: the same choices and weights, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(E)
    l = torch.randn(6000, E, device="cuda", generator=g)
    b = 0.2 * torch.randn(E, device="cuda", generator=g)
    kw = dict(score="sigmoid", groups=groups, top_groups=top, bias=b)
    w, e = X.route(l, 3, **kw)
    for r in (slice(0, 40), slice(5960, 6000)):
        w2, e2 = X.route(l[r], 3, **kw)
        assert torch.equal(e[r], e2) and (w[r] - w2).abs().max() <= 3e-7     # sums over slots in another order


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,k,groups,top", [(128, 8, 8, 4), (128, 5, 8, 2), (256, 8, 8, 4), (64, 6, 4, 2), (96, 7, 8, 3),
                                            (32, 4, 4, 2), (160, 3, 5, 2), (128, 32, 1, 1), (100, 9, 1, 1), (48, 2, 4, 2),
                                            (128, 1, 8, 4), (12, 5, 1, 1), (512, 8, 16, 8)])
def test_route_many_tokens_with_ties_and_closed_experts(E, k, groups, top, biased, dt):
    """Logits of few values: whole lanes of equal keys, groups of equal value, closed experts and NaN among them; the same
    200 rows over and over, more than a pass of the grid."""
    g = _gen(E * k + groups)
    l = torch.randint(-2, 3, (200, E), generator=g).double() / 2
    l[50:120] = l[50:120].masked_fill(torch.rand(70, E, generator=g) < 0.5, float("-inf"))
    l[120:150] = l[120:150].masked_fill(torch.rand(30, E, generator=g) < 0.97, float("-inf"))
    l[150:160] = 0.5
    l[160] = float("-inf")
    l[161, E // 2:] = float("-inf")
    l[162, E // 3] = float("inf")
    l = l.to(DT[dt])
    # biases that are multiples of an eighth: a biased sigmoid ties where logit and bias are equal, and is apart elsewhere
    b = torch.randint(-1, 2, (E,), generator=g).float() / 8 if biased else None
    kw = dict(score="sigmoid", groups=groups, top_groups=top)
    w, e = X.route(l.cuda().repeat(50, 1), k, bias=_cuda(b), **kw)
    w, e = w.cpu().view(50, 200, k), e.cpu().long().view(50, 200, k)
    assert torch.equal(e, e[:1].expand_as(e)) and torch.equal(w, w[:1].expand_as(w))
    w0, e0, gap = R.route(l, k, b, **kw)
    clear = (gap > 1e-6) | (gap == 0)             # equal values are equal in any arithmetic: they come from equal inputs
    assert clear.double().mean() > 0.9
    assert torch.equal(e[0][clear], e0[clear])
    assert (w[0].double() - w0)[clear].abs().max() <= 2e-6
    l[170:180, ::7] = float("nan")                # NaN ranks first, in order
    _, e = X.route(l[170:180].cuda().repeat(600, 1), k, score="sigmoid")
    first = torch.arange(0, E, 7)[:k]
    assert (e.cpu().long()[:, :len(first)] == first).all()


@pytest.mark.parametrize("T", [0, 1, 7, 5000])
def test_route_sizes_and_strides(T):
    g = _gen(T)
    wide = torch.randn(T, 100, generator=g)
    l = wide[:, 7:71]
    w, e = X.route(wide.cuda()[:, 7:71], 4)
    assert w.shape == (T, 4) and e.shape == (T, 4)
    if T:
        top = torch.topk(l, 4, dim=1)
        assert torch.equal(e.cpu().long(), top.indices)
        assert (w.cpu() - torch.softmax(top.values, 1)).abs().max() < 1e-6


def test_route_ties_nan_and_infinities():
    inf, nan = float("inf"), float("nan")
    l = torch.tensor([[1.0, 3.0, 3.0, 3.0], [0.0, -0.0, 0.0, -0.0], [1.0, nan, 2.0, nan], [-inf, -inf, 5.0, -inf],
                      [inf, 1.0, inf, 0.0], [-200.0, -300.0, -inf, -250.0]])
    w, e = X.route(l.cuda(), 2, score="sigmoid")
    assert e.cpu().tolist() == [[1, 2], [0, 1], [1, 3], [2, -1], [0, 2], [0, 3]]
    w = w.cpu()
    assert torch.isnan(w[2]).all() and w[3].tolist() == [1.0, 0.0] and w[4].tolist() == [0.5, 0.5]
    assert w[5].tolist() == [0.0, 0.0]            # both scores underflow: their sum is zero
    w, e = X.route(l.cuda(), 2)
    assert e.cpu().tolist() == [[1, 2], [0, 1], [1, 3], [2, -1], [0, 2], [0, 3]]
    w = w.cpu()
    assert w[5, 0] == 1.0 and abs(float(w[5, 1]) / math.exp(-50.0) - 1) < 1e-6
    assert torch.isnan(w[2]).all() and torch.isnan(w[4]).all()


def test_route_refusals():
    l = torch.randn(4, 12, device="cuda")
    for bad, msg in [(lambda: X.route(l, 0), "k must be"), (lambda: X.route(l, 13), "k must be"),
                     (lambda: X.route(l.double(), 2), "float32, bfloat16 or float16"),
                     (lambda: X.route(l, 2, groups=5), "do not split"),
                     (lambda: X.route(l, 2, groups=4, top_groups=5), "top_groups"),
                     (lambda: X.route(l, 2, bias=torch.zeros(11, device="cuda")), "bias must be"),
                     (lambda: X.route(l.view(2, 2, 12), 2), "\\[tokens, experts\\]"),
                     (lambda: X.route(torch.randn(2, 600, device="cuda"), 2), "at most 512"),
                     (lambda: X.route(l.cpu(), 2), "CUDA|backend")]:
        with pytest.raises((RuntimeError, NotImplementedError), match=msg):
            bad()
    with pytest.raises(ValueError, match="softmax"):
        X.route(l, 2, score="tanh")


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("T,k,E", [(0, 1, 3), (1, 1, 1), (5, 3, 2), (64, 8, 64), (1000, 2, 89), (8192, 1, 256), (8193, 1, 256),
                                   (5000, 2, 1000), (30000, 4, 16), (300000, 4, 20), (4097, 1, 3),
                                   (1050000, 1, 7)])
def test_plan_sorts_the_slots(T, k, E):
    g = _gen(T + E)
    ex = torch.randint(-1, E, (T, k), generator=g)
    if T > 100:
        ex[ex == E // 2] = -1                     # an expert without slots
    p = X.plan_experts(ex.cuda(), E)
    words = p.words.cpu()
    p.check()
    cnt = torch.bincount(ex[ex >= 0], minlength=E)
    seg = torch.zeros(E + 1, dtype=torch.int64)
    seg[1:] = torch.cumsum((cnt + 127) // 128 * 128, 0)
    assert int(words[0]) == int(seg[-1]) // 128
    o = 8
    assert torch.equal(words[o:o + E + 1].long(), seg)
    pairs = [int(seg[e]) // 128 + 2 * i for e in range(E) for i in range((int(seg[e + 1] - seg[e]) // 128 + 1) // 2)]
    assert int(words[2]) == len(pairs)
    assert torch.equal(words[o + E + 1:o + 2 * E + 1].long(), cnt)
    tiles = T * k // 128 + min(T * k, E)
    o_order, o_tile, o_row = o + 2 * E + 1, o + 3 * E + 1, o + 3 * E + 1 + 2 * tiles
    assert words[o_order:o_order + E].tolist() == sorted(range(E), key=lambda e: (-int(cnt[e]), e))
    rows = words[o_row:o_row + int(seg[-1])].long()
    want = torch.full((int(seg[-1]),), -1, dtype=torch.int64)
    flat = ex.reshape(-1)
    assert words[o_tile + tiles:o_tile + tiles + len(pairs)].tolist() == pairs
    for e in range(E):
        s = torch.nonzero(flat == e)[:, 0]
        want[seg[e]:seg[e] + len(s)] = s          # stable
        assert (words[o_tile + seg[e] // 128:o_tile + seg[e + 1] // 128] == e).all()
    assert torch.equal(rows, want)
    slot_row = words[o_row + tiles * 128:o_row + tiles * 128 + T * k].long()
    back = torch.full((T * k,), -1, dtype=torch.int64)
    at = torch.nonzero(want >= 0)[:, 0]
    back[want[at]] = at
    assert torch.equal(slot_row, back)


def test_plan_status_and_refusals():
    p = X.plan_experts(torch.tensor([[0, 3], [1, -2]], device="cuda"), 3)
    with pytest.raises(RuntimeError, match="outside"):
        p.check()
    x, w = torch.randn(2, 16, device="cuda"), torch.randn(3, 8, 16, device="cuda")
    want = torch.zeros(2, 2, 8, device="cuda")
    want[0, 0], want[1, 0] = w[0] @ x[0], w[1] @ x[1]
    for few in (True, False):                     # bad indices count as no expert in both forms
        got = N.ops().expert_linear(x, w, p.experts, None if few else p.words, None)
        assert (got - want).abs().max() < 1e-5
    with pytest.raises(ValueError, match="integer"):
        X.plan_experts(torch.zeros(3, 2), 4)
    with pytest.raises(RuntimeError, match="n_experts"):
        X.plan_experts(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 5000).words


# ------------------------------------------------------------------------------------------------ products
def _x_close(got, want, K, dt, roundings):
    val, mag = want
    assert got.shape == val.shape and got.dtype == dt
    tol = (8 + K / 8) * E32 * mag + U[dt] * val.abs() + (roundings * U[dt]) * mag
    if dt == torch.float16:
        tol = tol + 2.0 ** -24                    # half a step of the subnormals
    off = (got.double().cpu() - val).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {(off / (tol + 1e-300)).max()}"


def _x_inputs(T, k, E, D, O, dt, slots, g, skew=True):
    x = torch.randn(*((T, k, D) if slots else (T, D)), generator=g).to(dt)
    w = (torch.randn(E, O, D, generator=g) / math.sqrt(D)).to(dt)
    ex = torch.randint(0, E, (T, k), generator=g)
    if skew:
        ex[torch.rand(T, k, generator=g) < 0.4] = E // 2
        ex[torch.rand(T, k, generator=g) < 0.1] = -1
    p = torch.rand(T, k, generator=g) + 0.1
    return x, w, ex.to(torch.int32), p


PRODUCTS = [  # T, k, E, D, O
    (1, 1, 1, 8, 8), (3, 2, 4, 64, 64), (40, 2, 3, 64, 128), (130, 1, 2, 128, 256), (70, 4, 5, 200, 136), (33, 3, 7, 72, 515),
    (150, 2, 2, 129, 67), (20, 2, 3, 1, 1), (64, 2, 40, 24, 40), (300, 1, 3, 320, 264), (17, 8, 8, 65, 300),
]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,k,E,D,O", PRODUCTS)
@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_expert_linear_forward_and_backward(T, k, E, D, O, dt, slots, weighted):
    dt = DT[dt]
    g = _gen(T + D)
    x, w, ex, p = _x_inputs(T, k, E, D, O, dt, slots, g)
    p = p if weighted else None
    dy = torch.randn(*((T, O) if weighted else (T, k, O)), generator=g).to(dt)
    out0, dx0, dw0, dg0 = R.expert_linear(x, w, ex, p, dy)
    xd, wd, pd = _cuda(x, True), _cuda(w, True), _cuda(p, weighted)
    plan = X.plan_experts(ex.cuda(), E)
    out = X.expert_linear(xd, wd, plan, pd)
    _x_close(out.detach(), out0, D, dt, 1 if weighted and k > 1 else 0)
    ins = (xd, wd, pd) if weighted else (xd, wd)
    grads = torch.autograd.grad(out, ins, dy.cuda())
    _x_close(grads[0], dx0, O, dt, 1 if not slots and k > 1 else 0)
    _x_close(grads[1], dw0, T * k, dt, 1 if weighted else 0)
    if weighted:
        _x_close(grads[2], dg0, D + O, torch.float32, 0)
    few = N.ops().expert_linear(x.cuda(), w.cuda(), plan.experts, None, _cuda(p))
    _x_close(few, out0, D, dt, 0)
    plan.check()
    again = torch.autograd.grad(X.expert_linear(xd, wd, plan, pd), ins, dy.cuda())
    assert all(torch.equal(a, b) for a, b in zip(grads, again))            # fixed order of the sums


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (True, True, False)])
def test_expert_linear_gradients_one_at_a_time(need):
    g = _gen(9)
    x, w, ex, p = _x_inputs(50, 2, 4, 96, 40, torch.bfloat16, False, g)
    dy = torch.randn(50, 40, generator=g).bfloat16().cuda()
    plan = X.plan_experts(ex.cuda(), 4)
    full = [_cuda(t, True) for t in (x, w, p)]
    want = torch.autograd.grad(X.expert_linear(full[0], full[1], plan, full[2]), full, dy)
    part = [_cuda(t, n) for t, n in zip((x, w, p), need)]
    ins = [t for t, n in zip(part, need) if n]
    got = torch.autograd.grad(X.expert_linear(part[0], part[1], plan, part[2]), ins, dy)
    for a, b in zip(got, [t for t, n in zip(want, need) if n]):
        assert torch.equal(a, b)


def test_expert_linear_more_tiles_than_sms():
    """Every persistent CTA runs several tiles: ring phases and both accumulators wrap; checked against torch in fp64."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T, k, E, D, O = 20000, 2, 6, 192, 600
    x = torch.randn(T, D, device="cuda", generator=g).bfloat16()
    w = (torch.randn(E, O, D, device="cuda", generator=g) / 14).bfloat16()
    ex = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    p = torch.rand(T, k, device="cuda", generator=g)
    dy = torch.randn(T, O, device="cuda", generator=g).bfloat16()
    ins = [x.requires_grad_(), w.requires_grad_(), p.requires_grad_()]
    plan = X.plan_experts(ex, E)
    out = X.expert_linear(x, w, plan, p)
    dx, dw, dp = torch.autograd.grad(out, ins, dy)
    plan.check()
    ref = [t.detach().double().requires_grad_() for t in ins]
    z = torch.zeros(T, O, dtype=torch.float64, device="cuda")
    for e in range(E):
        for j in range(k):
            t = torch.nonzero(ex[:, j] == e)[:, 0]
            z = z.index_add(0, t, ref[2][t, j, None] * (ref[0][t] @ ref[1][e].T))
    want = (z, *torch.autograd.grad(z, ref, dy.double()))
    for a, b, n in zip((out, dx, dw, dp), want, (1.5, 1.5, 1.5, 0)):
        # random roundings: the 2-norm error of each is u / sqrt(3) relative; 1.5 covers the two of a sum over choices
        rel = float((a.detach().double() - b).norm() / b.norm())
        assert rel <= (n * U[torch.bfloat16] / math.sqrt(3) if n else 2e-6), rel


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_expert_linear_long_sums_keep_fp32_accuracy(dt):
    """The tensor cores truncate when they accumulate (about 1.7e-8 of the sum for each 16 terms), so long sums whose
    result leaves in fp32 are cut into chunks of 512: 32 x 1.7e-8 = 5.4e-7, and 1e-6 with the roundings of the rest.
    One accumulator over 2048 terms would be 2.2e-6 off, over 6000 6.4e-6."""
    g = torch.Generator(device="cuda").manual_seed(2)
    dt = DT[dt]
    T, D, O = 6000, 1024, 2048
    x = torch.randn(T, D, device="cuda", generator=g).to(dt).requires_grad_()
    w = (torch.randn(1, O, D, device="cuda", generator=g) / 32).to(dt).requires_grad_()
    p = torch.rand(T, 1, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(T, O, device="cuda", generator=g).to(dt)
    plan = X.plan_experts(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), 1)
    out = X.expert_linear(x, w, plan, p)
    dx, dw, dp = torch.autograd.grad(out, (x, w, p), dy)
    plan.check()
    z = x.detach().double() @ w.detach()[0].double().T
    dz = p.detach().double() * dy.double()
    want = {"dp": (dy.double() * z).sum(1, keepdim=True)}
    got = {"dp": dp}
    if dt == torch.float32:
        want |= {"out": p.detach().double() * z, "dx": dz @ w.detach()[0].double(), "dw": (dz.T @ x.detach().double())[None]}
        got |= {"out": out.detach(), "dx": dx, "dw": dw}
    for n in want:
        rel = float((got[n].double() - want[n]).norm() / want[n].norm())
        assert rel <= 1e-6, (n, rel)


def test_expert_linear_padding_rows_do_not_spread_nan():
    """A NaN in one atom's row reaches that atom's output and its experts' gradients only."""
    g = _gen(11)
    for dt in (torch.float32, torch.bfloat16):
        x, w, ex, p = _x_inputs(60, 2, 5, 64, 48, dt, False, g, skew=False)
        ex[0] = torch.tensor([0, 1], dtype=torch.int32)
        ex[1:] = torch.randint(2, 5, (59, 2), generator=g, dtype=torch.int32)
        x[0, 3] = float("nan")
        xd, wd = _cuda(x, True), _cuda(w, True)
        out = X.expert_linear(xd, wd, X.plan_experts(ex.cuda(), 5), p.cuda())
        dx, dw = torch.autograd.grad(out, (xd, wd), torch.ones_like(out))
        assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()
        assert torch.isnan(dw[:2, :, 3]).all() and torch.isfinite(dw[2:]).all() and torch.isfinite(dx).all()


def test_expert_linear_bad_gradients_stay_in_their_experts():
    """NaN and infinities in one token's upstream gradient reach its dx, its dweights and its experts' dW only."""
    g = _gen(14)
    for dt in (torch.float32, torch.bfloat16):
        for bad in (float("nan"), float("inf")):
            x, w, ex, p = _x_inputs(200, 2, 5, 64, 48, dt, False, g, skew=False)
            ex[0] = torch.tensor([0, 1], dtype=torch.int32)
            ex[1:] = torch.randint(2, 5, (199, 2), generator=g, dtype=torch.int32)
            ex[50:90, 0] = 0
            xd, wd, pd = _cuda(x, True), _cuda(w, True), _cuda(p, True)
            dy = torch.randn(200, 48, generator=g).to(dt)
            dy[0, 5] = bad
            out = X.expert_linear(xd, wd, X.plan_experts(ex.cuda(), 5), pd)
            dx, dw, dp = torch.autograd.grad(out, (xd, wd, pd), dy.cuda())
            assert not torch.isfinite(dx[0]).any() and torch.isfinite(dx[1:]).all()
            assert not torch.isfinite(dp[0]).any() and torch.isfinite(dp[1:]).all()
            assert not torch.isfinite(dw[:2, 5]).any() and torch.isfinite(dw[2:]).all()
            rest = [o for o in range(48) if o != 5]
            assert torch.isfinite(dw[:2, rest]).all()


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), 3.4e38])
def test_expert_linear_infinities_stay_in_their_rows(bad):
    """Infinite values (and, in fp32, values that the first bfloat16 plane rounds to infinity) leave every other row alone."""
    g = _gen(12)
    for dt in (torch.float32, torch.bfloat16):
        x, w, ex, p = _x_inputs(60, 2, 5, 64, 48, torch.float32, False, g, skew=False)
        x, w = x.to(dt), w.to(dt)
        x[7, 3] = bad
        plan = X.plan_experts(ex.cuda(), 5)
        out = N.ops().expert_linear(x.cuda(), w.cuda(), plan.experts, plan.words, p.cuda())
        others = torch.arange(60) != 7
        if math.isinf(bad):
            assert not torch.isfinite(out[7]).any()
        x[7, 3] = 0.0
        want = N.ops().expert_linear(x.cuda(), w.cuda(), plan.experts, plan.words, p.cuda())
        assert torch.equal(out[others.cuda()], want[others.cuda()])


def test_offsets_beyond_32_bits():
    """Outputs of more than 2^31 elements: the last rows equal those of a call on the last rows alone."""
    g = torch.Generator(device="cuda").manual_seed(3)
    T, D, O = 1_100_000, 64, 2048
    x = torch.randn(T, D, device="cuda", generator=g).bfloat16()
    w = torch.randn(2, O, D, device="cuda", generator=g).bfloat16() / 8
    ex = torch.randint(0, 2, (T, 1), device="cuda", generator=g, dtype=torch.int32)
    plan = N.ops().expert_plan(ex, 2)
    y = N.ops().expert_linear(x, w, ex, plan, None)[:, 0]
    assert y.numel() > 2 ** 31
    tail = N.ops().expert_linear(x[-300:], w, ex[-300:].contiguous(), N.ops().expert_plan(ex[-300:].contiguous(), 2), None)
    assert torch.equal(y[-300:], tail[:, 0])
    n, m, r = N.ops().layer_norm_fwd(y, None, None, 1e-5)
    n2, m2, r2 = N.ops().layer_norm_fwd(y[-300:].clone(), None, None, 1e-5)
    assert torch.equal(n[-300:], n2) and torch.equal(m[-300:], m2) and torch.equal(r[-300:], r2)
    dx, _, _ = N.ops().layer_norm_bwd(y, n, None, m, r, True, False, False, False)
    d2, _, _ = N.ops().layer_norm_bwd(y[-300:].clone(), n2, None, m2, r2, True, False, False, False)
    assert torch.equal(dx[-300:], d2)
    dy = y[:, None]
    dxx, dww, _ = N.ops().expert_linear_bwd(dy, x, w, ex, plan, None, True, True, False)
    tdx, _, _ = N.ops().expert_linear_bwd(dy[-300:], x[-300:], w, ex[-300:].contiguous(),
                                          N.ops().expert_plan(ex[-300:].contiguous(), 2), None, True, False, False)
    assert torch.equal(dxx[-300:], tdx) and torch.isfinite(dww).all()
    del n, dx, dy, dxx
    l = y.view(-1)[:2 ** 31 + 2 ** 20].view(-1, 512)
    wt, e = N.ops().route(l, None, 2, True, 1, 1, True, 1.0)
    wt2, e2 = N.ops().route(l[-40:].clone(), None, 2, True, 1, 1, True, 1.0)
    assert torch.equal(e[-40:], e2) and torch.allclose(wt[-40:], wt2, rtol=1e-6)
    dl = N.ops().route_bwd(wt, l, e, True, True, 1.0)
    assert torch.equal(dl[-40:], N.ops().route_bwd(wt[-40:].contiguous(), l[-40:].clone(), e2, True, True, 1.0))


@pytest.mark.parametrize("T,D,O", [(300, 64, 64), (40000, 1024, 1024)])
def test_expert_linear_timeout_path_reports_and_recovers(T, D, O):
    """The bounded waits, driven from the host: with one load withheld they run out after 20 ms, the kernel drains, frees
    its TMEM and reports; the next launch with the default limit is right.  The larger size runs on pairs of CTAs."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(T, D, device="cuda", generator=g).bfloat16()
    w = (torch.randn(1, O, D, device="cuda", generator=g) / math.sqrt(D)).bfloat16()
    plan = X.plan_experts(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), 1)
    plan.check()
    try:
        N.check(N.lib().mace_b200_expert_test_hooks(20_000_000, 1), "expert_test_hooks")
        N.ops().expert_linear(x, w, plan.experts, plan.words, None)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="gave up waiting"):
            plan.check()
    finally:
        N.check(N.lib().mace_b200_expert_test_hooks(2_000_000_000, 0), "expert_test_hooks")
    plan = X.plan_experts(plan.experts, 1)
    out = N.ops().expert_linear(x, w, plan.experts, plan.words, None)[:, 0]
    plan.check()
    want = x.double() @ w[0].double().T
    assert float((out.double() - want).norm() / want.norm()) <= U[torch.bfloat16] / math.sqrt(3)


def test_expert_linear_empty_and_unrouted():
    w = torch.randn(3, 8, 16, device="cuda", requires_grad=True)
    x = torch.randn(0, 16, device="cuda", requires_grad=True)
    plan = X.plan_experts(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 3)
    out = X.expert_linear(x, w, plan, torch.zeros(0, 2, device="cuda"))
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert out.shape == (0, 8) and dx.shape == (0, 16) and dw.shape == w.shape and not dw.any()
    x = torch.randn(70, 16, device="cuda", requires_grad=True)
    plan = X.plan_experts(torch.full((70, 2), -1, device="cuda"), 3)
    p = torch.rand(70, 2, device="cuda", requires_grad=True)
    out = X.expert_linear(x, w, plan, p)
    grads = torch.autograd.grad(out.sum(), (x, w, p))
    assert not out.any() and not any(t.any() for t in grads)


def test_expert_linear_strided_rows_and_side_stream():
    """Rows of [n, 4, 128] features read in place; a call on a stream of its own is ordered like any torch operation."""
    g = _gen(13)
    h = torch.randn(90, 4, 128, generator=g)
    w = torch.randn(4, 56, 128, generator=g) / 11.3
    ex = torch.randint(0, 4, (90, 2), generator=g, dtype=torch.int32)
    p = torch.rand(90, 2, generator=g)
    out0, outa = R.expert_linear(h[:, 2], w, ex, p)
    hd, wd, exd, pd = h.cuda(), w.cuda(), ex.cuda(), p.cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = X.expert_linear(hd[:, 2], wd, X.plan_experts(exd, 4), pd)
    side.synchronize()
    _x_close(out, (out0, outa), 128, torch.float32, 1)


def test_expert_linear_gradient_against_differences():
    g = _gen(15)
    x, w, ex, p = _x_inputs(12, 2, 3, 20, 10, torch.float32, False, g)
    dy = torch.randn(12, 10, generator=g)
    ins = [_cuda(t, True) for t in (x, w, p)]
    grads = torch.autograd.grad(X.expert_linear(ins[0], ins[1], X.plan_experts(ex.cuda(), 3), ins[2]), ins, dy.cuda())
    h = 1e-5
    for i, gr in enumerate(grads):
        v = torch.randn(gr.shape, generator=g, dtype=torch.float64)
        args = [t.double() for t in (x, w, p)]
        f = []
        for s in (1, -1):
            q = [a + s * h * v if n == i else a for n, a in enumerate(args)]
            f.append((R.expert_linear(q[0], q[1], ex, q[2])[0] * dy.double()).sum())
        fd = float((f[0] - f[1]) / (2 * h))
        assert abs(float((gr.double().cpu() * v).sum()) - fd) <= 2e-5 * (1 + abs(fd))


def test_expert_linear_refusals():
    x, w = torch.randn(6, 16, device="cuda"), torch.randn(3, 8, 16, device="cuda")
    ex = torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    plan, p = X.plan_experts(ex, 3), torch.rand(6, 2, device="cuda")
    for bad, msg in [(lambda: X.expert_linear(x[:, :8], w, plan), "x must be"),
                     (lambda: X.expert_linear(x[:5], w, plan), "x must be"),
                     (lambda: X.expert_linear(x.bfloat16(), w, plan), "differ in type"),
                     (lambda: X.expert_linear(x.double(), w.double(), plan), "float32, bfloat16 or float16"),
                     (lambda: X.expert_linear(x, w, plan, p[:, :1]), "weights must be"),
                     (lambda: X.expert_linear(x, w, plan, p.bfloat16()), "weights must be"),
                     (lambda: X.expert_linear(x, w.cpu(), plan), "CUDA tensor"),
                     (lambda: X.expert_linear(x.view(6, 1, 16), w, plan), "x must be"),
                     (lambda: N.ops().expert_linear(x, w, ex, plan.words[:-1].contiguous(), None), "does not belong")]:
        with pytest.raises(RuntimeError, match=msg):
            bad()
    with pytest.raises(ValueError, match="w must be"):
        X.expert_linear(x, w[:2], plan)
    with pytest.raises(TypeError, match="ExpertPlan"):
        X.expert_linear(x, w, ex)


# ------------------------------------------------------------------------------------------------ together
def test_expert_block_matches_the_fp64_forms():
    g = _gen(21)
    T, D, F, O, E, k = 45, 96, 40, 24, 6, 2
    block = X.ExpertBlock(D, F, O, E, k, seed=3)
    x = torch.randn(T, 4, D, generator=g)
    dy = torch.randn(T, O, generator=g)
    xd = _cuda(x, True)
    out = block(xd[:, 1])
    names = ["gamma", "beta", "router", "w1", "w2"]
    grads = torch.autograd.grad(out, [xd] + [getattr(block, n) for n in names], dy.cuda())
    p = {n: getattr(block, n).detach().double().cpu().requires_grad_() for n in names}
    x64 = x.double().requires_grad_()
    xs = x64[:, 1]
    c = xs - xs.mean(1, keepdim=True)
    xn = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * p["gamma"] + p["beta"]
    ex = block.plan.experts.cpu().long()
    w = R.route_weights(xn @ p["router"].T, ex, "sigmoid")
    h = torch.nn.functional.silu(torch.einsum("td,tkfd->tkf", xn, p["w1"][ex]))
    ref = (w[..., None] * torch.einsum("tkf,tkof->tko", h, p["w2"][ex])).sum(1)
    want = torch.autograd.grad(ref, [x64] + [p[n] for n in names], dy.double())
    assert (out.detach().double().cpu() - ref).abs().max() <= 2e-5 * ref.abs().max()
    for a, b in zip(grads, want):
        # a chain of six fp32 operators, each within a few 1e-7 of its largest value
        assert (a.double().cpu() - b).abs().max() <= 2e-5 * b.abs().max()
    load = block.balance(0.5)
    assert int(load.sum()) == T * k and torch.equal(block.bias.cpu(), 0.5 * torch.sign(load.mean() - load).cpu())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_train_readout_learns(dt):
    r = X.train_readout(n=4, n_experts=4, k=2, hidden=32, steps=60, dtype=DT[dt])
    assert r["atoms"] == 192 and sum(r["load"]) == 384
    assert r["loss_last"] < 0.5 * r["loss_first"]


def test_experts_command_line(capsys, monkeypatch):
    import json

    monkeypatch.setattr("sys.argv", ["experts", "--n", "4", "--steps", "3", "--experts", "5", "--k", "1"])
    X.main()
    assert json.loads(capsys.readouterr().out)["experts"] == 5


def test_operators_replay_in_a_cuda_graph():
    """No call synchronises or depends on values read back: the whole chain is capturable, and a replay follows new inputs."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(300, 64, device="cuda", generator=g)
    gamma, wr = torch.ones(64, device="cuda"), torch.randn(8, 64, device="cuda", generator=g)
    w = torch.randn(8, 72, 64, device="cuda", generator=g) / 8

    def chain():
        xn = X.layer_norm(x, gamma)
        wts, ex = X.route(xn @ wr.T, 2)
        return N.ops().expert_linear(xn, w, ex, N.ops().expert_plan(ex, 8), wts)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = chain()
    for seed in (6, 7):
        x.copy_(torch.randn(300, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, chain())
