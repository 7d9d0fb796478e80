"""Orthogonalised matrices (mace_onegpu.optim.orthogonalize, Muon) against the plain fp64 form: shapes wide, tall, odd, single rows and
columns, batches, strides, types; gradients of low rank and of wide spectra; zero matrices, non-finite values, refusals.

Tolerances (Frobenius norm of the difference over that of the result).  The rounding to bf16 is at most 2^-8 of an element.  Before
it: each of the steps rounds two left factors to fp16 (2^-11 of their off-diagonal entries) and reads fp16 products' operands
(2^-11), and the polynomial's slope is up to 3.4 near the singular values that a step leaves at 0.7 to 1.2, so the errors of
`steps` steps in 3 places come to at most 3 steps 2^-11 in the worst case, and about the root of that many independent ones in
the mean: sqrt(15) 2^-11 = 1.9e-3."""
import pytest
import torch

from mace_onegpu import optim as X

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOL = 2.0 ** -8 + 15 * 2.0 ** -11 / 2     # one rounding in full and half of the worst case of the others: 7.6e-3


def plain(g, steps=5, coef=X.COEFFICIENTS, eps=1e-7):
    x = g.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    rows = coef if isinstance(coef[0], (tuple, list)) else [coef] * steps
    for a, b, c in rows:
        if g.shape[-2] <= g.shape[-1]:
            s = x @ x.mT
            x = a * x + (b * s + c * s @ s) @ x
        else:
            s = x.mT @ x
            x = a * x + x @ (b * s + c * s @ s)
    return x


def _rel(u, want):
    d = (u.double() - want).flatten(-2).norm(dim=-1) / want.flatten(-2).norm(dim=-1)
    return float(d.max())


SHAPES = [(1, 1, 1), (1, 1, 50), (1, 50, 1), (2, 3, 5), (3, 16, 16), (1, 64, 128), (8, 64, 128), (2, 128, 64), (5, 100, 333),
          (4, 333, 100), (89, 128, 512), (20, 512, 128), (1, 129, 129), (3, 515, 1023), (2, 1023, 515), (1, 1000, 4096), (1, 4096, 1000),
          (1, 2048, 2048), (300, 24, 40), (1, 260, 20000), (1, 20000, 200)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,m,n", SHAPES)
def test_random_matrices(b, m, n, dt):
    g = (torch.randn(b, m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(m + n)) * 3).to(DT[dt])
    u = X.orthogonalize(g)
    assert u.dtype == torch.bfloat16 and u.shape == g.shape
    assert _rel(u, plain(g)) < TOL
    assert torch.equal(u, X.orthogonalize(g))


@pytest.mark.parametrize("m,n", [(200, 300), (768, 512), (1024, 1024)])
def test_spectra(m, n):
    """Decaying spectra and low rank over noise: errors added to weak directions would grow 485-fold."""
    gen = torch.Generator("cuda").manual_seed(m)

    def rnd(*s):
        return torch.randn(*s, device="cuda", generator=gen)

    k = min(m, n)
    u, v = torch.linalg.qr(rnd(m, k))[0], torch.linalg.qr(rnd(n, k))[0]
    cases = [u * torch.logspace(0, -5, k, device="cuda") @ v.T, rnd(m, 8) @ rnd(8, n) + 1e-3 * rnd(m, n), rnd(m, 1) @ rnd(1, n),
             rnd(m, 8) @ rnd(8, n), u @ v.T]
    for i, g in enumerate(cases):
        assert _rel(X.orthogonalize(g * 1e-3), plain(g * 1e-3)) < TOL, i
    s = torch.linalg.svdvals(X.orthogonalize(cases[4]).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


def test_scales_and_steps():
    g = torch.randn(3, 70, 90, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    for scale in (1e-30, 1e-6, 1e18, 1e30):
        assert _rel(X.orthogonalize(g * scale), plain(g * scale)) < TOL
    # far below eps X = g 1e-30 / 1e-7, whose squares vanish: each step multiplies by a, 3.4445^5 = 484.9
    assert float(X.orthogonalize(g * 1e-30).abs().max()) < 485e-23 * (1 + 2.0 ** -8) * float(g.abs().max())
    assert _rel(X.orthogonalize(g * 1e-30, eps=1e-30), plain(g * 1e-30, eps=1e-30)) < TOL
    for steps in (1, 2, 7, 16):
        assert _rel(X.orthogonalize(g, steps=steps), plain(g, steps)) < TOL * max(1, steps / 5)
    rows = ((2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (3.0, -3.2, 1.2))
    assert _rel(X.orthogonalize(g, steps=3, coefficients=rows), plain(g, 3, rows)) < TOL


def test_strides_batches_and_single():
    g = torch.randn(4, 6, 40, 56, device="cuda")
    u = X.orthogonalize(g)
    assert u.shape == g.shape and _rel(u, plain(g)) < TOL
    for i in (0, 3):
        assert torch.equal(X.orthogonalize(g[i, 2]), u[i, 2])
    assert torch.equal(X.orthogonalize(g[:, 1]), u[:, 1])                    # batch stride
    wide = torch.randn(40, 100, device="cuda")
    assert torch.equal(X.orthogonalize(wide[:, 7:63]), X.orthogonalize(wide[:, 7:63].contiguous()))
    t = X.orthogonalize(g[0, 0].T)
    assert _rel(t, plain(g[0, 0].T)) < TOL
    one = torch.randn(40, 56, device="cuda")
    assert torch.equal(X.orthogonalize(one.expand(3, 40, 56))[2], X.orthogonalize(one))
    assert X.orthogonalize(g[:0]).shape == (0, 6, 40, 56) and X.orthogonalize(g[0, 0, :0]).shape == (0, 56)


def test_zero_and_non_finite():
    g = torch.randn(4, 50, 80, device="cuda")
    want = X.orthogonalize(g)
    bad = g.clone()
    bad[1] = 0
    bad[2, 3, 4] = float("nan")
    bad[3, 0, 0] = float("inf")
    u = X.orthogonalize(bad)
    assert torch.equal(u[0], want[0]) and not u[1].any() and u[2].isnan().all() and u[3].isnan().all()


def test_refusals():
    g = torch.randn(8, 16, device="cuda")
    with pytest.raises(ValueError, match="steps"):
        X.orthogonalize(g, steps=0)
    with pytest.raises(ValueError, match="coefficients"):
        X.orthogonalize(g, steps=2, coefficients=((1.5, -0.5, 0.0),))
    with pytest.raises(RuntimeError, match="reaches"):
        X.orthogonalize(g, coefficients=(9.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="reaches"):
        X.orthogonalize(g, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(RuntimeError, match="eps"):
        X.orthogonalize(g, eps=0.0)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        X.orthogonalize(g.double())
    with pytest.raises(RuntimeError, match="must be"):
        X.orthogonalize(g[0])
    with pytest.raises(RuntimeError, match="no gradient"):
        X.orthogonalize(g.requires_grad_())
    with pytest.raises(ValueError, match="matrices"):
        X.Muon([torch.nn.Parameter(torch.zeros(3, device="cuda"))])


def test_streams_and_graphs():
    g = torch.randn(3, 200, 300, device="cuda")
    want = X.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = X.orthogonalize(g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = X.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want)
    g.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, -want)


@pytest.mark.parametrize("nesterov", [False, True])
def test_muon(nesterov):
    """Three steps against the same recurrences in fp64: an update is off by TOL of its norm."""
    gen = torch.Generator("cuda").manual_seed(1)
    shapes = [(4, 30, 20), (48, 64)]
    ps = [torch.nn.Parameter(torch.randn(*s, device="cuda", generator=gen)) for s in shapes]
    ref, vs = [p.detach().double() for p in ps], [torch.zeros(*s, device="cuda", dtype=torch.float64) for s in shapes]
    opt = X.Muon(ps, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.05)
    for step in range(3):
        for i, p in enumerate(ps):
            p.grad = torch.randn(*shapes[i], device="cuda", generator=gen)
            vs[i] = 0.9 * vs[i] + p.grad.double()
            u = plain(p.grad.double() + 0.9 * vs[i] if nesterov else vs[i])
            ref[i] = ref[i] * (1 - 0.1 * 0.05) - 0.1 * max(1.0, shapes[i][-2] / shapes[i][-1]) ** 0.5 * u
        opt.step()
    for p, r, s in zip(ps, ref, shapes):
        off = (p.detach().double() - r).flatten(-2).norm(dim=-1)
        assert (off < 3 * 0.1 * 1.3 * 1.3 * min(s[-2:]) ** 0.5 * TOL).all()
