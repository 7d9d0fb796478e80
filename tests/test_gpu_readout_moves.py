"""Int8Readout under the casts and moves of a module: the scales stay float32, rows of the matrices whole 16 bytes apart."""
import copy

import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu


def _served(seed=0):
    return X.ReadoutBlock(40, 30, 5, 2, seed=seed).quantized()   # neither width is a multiple of 16


def _plain(r, x, off):
    z = X.group_norm(x, r.groups, r.gamma1, r.beta1, activation="silu", offsets=off)
    h = X.int8_linear(z, r.wq1, r.ws1, r.b1)
    z = X.group_norm(h, r.groups, r.gamma2, r.beta2, activation="silu", offsets=off)
    return X.int8_linear(z, r.wq2, r.ws2, r.b2)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16().float(), lambda m: m.to("cuda", torch.float16),
                                  lambda m: m.cpu().cuda(), lambda m: m.half().cpu().to("cuda"), copy.deepcopy])
def test_casts_and_moves(cast):
    ref = _served()
    scales, weights = [ref.ws1.clone(), ref.ws2.clone()], [ref.wq1.clone(), ref.wq2.clone()]
    r = cast(ref)
    dt = r.gamma1.dtype
    assert torch.equal(r.ws1, scales[0]) and torch.equal(r.ws2, scales[1]) and r.ws1.dtype == torch.float32
    for q, w in zip((r.wq1, r.wq2), weights):
        assert torch.equal(q, w) and q.stride(0) % 16 == 0 and q.stride(1) == 1 and q.is_cuda
    x, off = torch.randn(70, 40, device="cuda").to(dt), torch.tensor([0, 30, 70]).cuda()
    y = r(x, off)
    assert y.dtype == dt and torch.equal(y, _plain(r, x, off)) and bool(y.isfinite().all())


def test_state_goes_into_another_module():
    a, b = _served(0), _served(1).cpu().cuda()
    b.load_state_dict(a.state_dict())
    x = torch.randn(70, 40, device="cuda")
    assert torch.equal(a(x), b(x)) and b.wq2.stride(0) == 32
