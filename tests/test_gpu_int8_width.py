"""Rows of the greatest width that quantize_rows takes, and 8-bit rows that lie further apart than 32 bits count: column counters do not
overflow.  Values are compared with the definition in fp64, ties to even."""
import pytest
import torch

from mace_onegpu import _native as N
from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu


def test_widest_row():
    """2^31 - 17 columns: a warp's step behind the last one leaves 31 bits (a warp goes over the row for some seconds)."""
    k = 2 ** 31 - 17
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(1, k, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    x[0, -1] = -9.0                                           # the largest is the last one
    q, s = X.quantize_rows(x)
    assert q.shape == (1, k) and float(s) == float(torch.tensor(9.0) / 127) and int(q[0, -1]) == -127
    scale, step = s.double(), 2 ** 28
    for lo in range(0, k, step):
        want = torch.round(x[0, lo:lo + step].double() / scale)
        assert torch.equal(q[0, lo:lo + step].double(), want), lo


def test_rows_far_apart():
    """The C ABI with rows of 20 values 2^31 + 8 bytes apart: the bytes between them are zeroed."""
    k, ld = 20, 2 ** 31 + 8
    x = torch.randn(2, k, device="cuda")
    q = torch.full((ld + k,), 1, device="cuda", dtype=torch.int8)
    s = torch.empty(2, device="cuda")
    # a row each, so that the buffer ends with the second one's values
    L, st = N.lib(), torch.cuda.current_stream().cuda_stream
    assert L.mace_b200_quantize_rows(x.data_ptr(), k, q.data_ptr(), ld, s.data_ptr(), 1, k, 0, st) == 0
    assert L.mace_b200_quantize_rows(x[1].data_ptr(), k, q.data_ptr() + ld, k, s[1:].data_ptr(), 1, k, 0, st) == 0
    torch.cuda.synchronize()
    want, ws = X.quantize_rows(x)
    assert torch.equal(q[:k], want[0]) and not q[k:ld].any() and torch.equal(q[ld:], want[1]) and torch.equal(s, ws)
