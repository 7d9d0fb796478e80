"""Orthogonalised matrices of few rows or of low rank over noise: what a step leaves in their weak directions grows by up to a^4 = 140
in the later ones, so an error there that is not proportional to the direction itself shows.

Tolerances (Frobenius norm of the difference over that of the result; TOL as in test_gpu_orth.py: one rounding to bfloat16 in full and
half of the worst case of 15 others of 2^-11).  The root mean square over a batch of matrices stays below TOL; a single matrix of a few
elements, where nothing averages out, below twice that, which is more than all of these roundings in full, 2^-8 + 15 2^-11 = 1.1e-2."""
import pytest
import torch

from mace_onegpu import optim as X
from test_gpu_orth import TOL, plain

pytestmark = pytest.mark.gpu

SHAPES = [(2, 2), (3, 3), (3, 5), (4, 64), (64, 4), (8, 64), (16, 16), (16, 128), (128, 16), (64, 128), (128, 700), (5, 3000), (3000, 5), (140, 140),
          (150, 400), (400, 150)]


@pytest.mark.parametrize("noise", [None, 0.1, 1e-2, 1e-3, 1e-4, 1e-6])
@pytest.mark.parametrize("m,n", SHAPES)
def test_low_rank_over_noise(m, n, noise):
    g = torch.Generator("cuda").manual_seed(m * n)
    batch = 200 if m * n < 20000 else 10
    for rank in (1, max(1, min(m, n) // 8), max(1, min(m, n) // 2)):
        x = torch.randn(batch, m, n, device="cuda", generator=g)
        if noise is not None:
            strong = torch.randn(batch, m, rank, device="cuda", generator=g) @ torch.randn(batch, rank, n, device="cuda", generator=g)
            x = strong + noise * x
        want = plain(x)
        off = (X.orthogonalize(x).double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
        assert float(off.square().mean().sqrt()) < TOL and float(off.max()) < 2 * TOL, (rank, float(off.max()))


def test_other_polynomials():
    """Steps that hardly grow, a single step, sixteen: each against fp64."""
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(50, 6, 1, device="cuda", generator=g) @ torch.randn(50, 1, 40, device="cuda", generator=g)
    x = x + 1e-3 * torch.randn(50, 6, 40, device="cuda", generator=g)
    for steps, coef in ((1, X.COEFFICIENTS), (2, X.COEFFICIENTS), (3, X.COEFFICIENTS), (8, (1.5, -0.5, 0.0)), (16, (1.5, -0.5, 0.0)),
                        (4, ((4.0, -6.0, 2.5), (3.0, -4.0, 1.5), (2.0, -1.5, 0.4), (1.5, -0.5, 0.0)))):
        want = plain(x, steps, coef)
        off = (X.orthogonalize(x, steps=steps, coefficients=coef).double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
        assert float(off.square().mean().sqrt()) < TOL and float(off.max()) < 2 * TOL, (steps, coef, float(off.max()))
