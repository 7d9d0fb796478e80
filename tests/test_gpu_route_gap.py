"""Renormalised softmax weights of experts that a bias, or the choice of groups, takes far below the row's largest logit: they
depend on the chosen logits alone, in the forward pass as in the gradient."""
import pytest
import torch

from mace_onegpu import experts as X

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [60.0, 95.0, 120.0, 1e4])
@pytest.mark.parametrize("T", [3, 9000])
def test_biased_softmax_far_below_the_row_maximum(gap, T):
    g = torch.Generator().manual_seed(int(gap))
    E, k = 24, 3
    l = torch.randn(T, E, generator=g)
    l[:, 5] += gap                                 # never chosen: its bias is low
    b = 0.01 * torch.randn(E, generator=g)
    b[5] = -5.0
    b[[2, 11, 17]] = torch.tensor([4.0, 3.0, 2.0])
    ld = l.cuda().requires_grad_()
    w, e = X.route(ld, k, bias=b.cuda(), score="softmax")
    assert (e.cpu() == torch.tensor([2, 11, 17])).all()
    sel = l.double()[:, [2, 11, 17]]
    want = torch.softmax(sel, 1)                   # the row's sum cancels
    assert (w.detach().double().cpu() - want).abs().max() <= 2e-6
    dw = torch.randn(T, k, generator=g)
    dl, = torch.autograd.grad(w, ld, dw.cuda())
    d0 = want * (dw.double() - (want * dw.double()).sum(1, keepdim=True))
    assert (dl.double().cpu()[:, [2, 11, 17]] - d0).abs().max() <= 2e-6 * dw.abs().max()
    rest = [i for i in range(E) if i not in (2, 11, 17)]
    assert not dl[:, rest].any()


@pytest.mark.parametrize("T", [3, 9000])
def test_grouped_softmax_far_below_the_row_maximum(T):
    """With a bias the best group need not hold the largest logit."""
    g = torch.Generator().manual_seed(2)
    E, k, groups = 32, 4, 4
    l = torch.randn(T, E, generator=g)
    l[:, 3] += 130.0
    b = torch.zeros(E)
    b[8:16] = 3.0                                  # group 1 wins whatever the scores
    w, e = X.route(l.cuda(), k, bias=b.cuda(), score="softmax", groups=groups, top_groups=1)
    e = e.cpu().long()
    assert ((e >= 8) & (e < 16)).all()
    want = torch.softmax(l.double().gather(1, e), 1)
    assert (w.double().cpu() - want).abs().max() <= 2e-6
