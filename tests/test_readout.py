"""Host side of group norm, products in 8-bit integers and orthogonalised matrices: argument checks of the C ABI and the Python modules
that come before any launch, shape functions, and the plain fp64 forms the GPU tests compare with, against torch's own
operations."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

import readout_refs as R
from mace_onegpu import _native as N
from mace_onegpu import experts, optim
from mace_onegpu import readout as X


def _error():
    return N.lib().mace_b200_last_error()


def test_bad_arguments_come_back_as_codes():
    L, n = N.lib(), N.c_i64()
    one = (ctypes.c_float * 4)()
    p = ctypes.addressof(one)
    gn = lambda rows, ns, ln, c, g, act=0, dt=0, pt=0, ld=None: L.mace_b200_group_norm_fwd(  # noqa: E731
        p, c if ld is None else ld, None, None, None, 0, p, None, None, None, rows, ns, ln, c, g, 1e-5, act, dt, pt, None)
    for bad in ((6, 2, 4, 8, 2), (6, 2, 3, 8, 3), (6, 2, 3, 8, 0), (-1, 2, 3, 8, 2), (6, 2, 3, 8, 2, 0, 0, 0, 7)):
        assert gn(*bad) < 0 and b"bad sizes" in _error(), bad
    assert gn(6, 2, 3, 8, 2, 9) < 0 and b"activation" in _error()
    assert gn(6, 2, 3, 8, 2, 0, 5) < 0 and b"types" in _error()
    assert gn(6, 2, 3, 8, 2, 0, 0, 1) < 0 and b"types" in _error()
    assert L.mace_b200_group_norm_workspace(6, 2, 4, 8, 2, 0, 0, 0, N.byref(n)) < 0 and b"bad sizes" in _error()

    assert L.mace_b200_quantize_rows(p, 8, p, 7, p, 3, 8, 0, None) < 0 and b"row strides" in _error()
    assert L.mace_b200_quantize_rows(p, 8, p, 16, p, 3, 8, 7, None) < 0 and b"type 7" in _error()
    assert L.mace_b200_quantize_rows(None, 8, None, 16, None, 0, 8, 0, None) == 0
    i8 = lambda t, k, nn, ldw=16, dt=0, bt=0, w=p: L.mace_b200_int8_linear(p, k, None, k, None, w, ldw, p, None, p, t, k, nn, dt, bt, None)  # noqa: E731
    for bad in ((-1, 8, 4), (3, 0, 4), (3, 8, 0), (3, 131072, 4, 131072), (3, 32, 4, 16), (3, 8, 4, 16, 8), (3, 8, 4, 16, 1, 2)):
        assert i8(*bad) < 0 and b"bad arguments" in _error(), bad
    assert i8(300, 8, 4) < 0 and b"null pointer" in _error()            # many tokens need buffers for their 8-bit form
    assert i8(1, 8, 4, 24) < 0 and b"16 bytes" in _error()
    assert i8(0, 8, 4) == 0
    assert L.mace_b200_int8_linear_few(1, 1024) == 1 and L.mace_b200_int8_linear_few(1000, 1024) == 0

    for b, m, k in ((-1, 4, 4), (65536, 4, 4), (1, 0, 4), (1, 4, 65537)):
        assert L.mace_b200_orthogonalize_workspace(b, m, k, N.byref(n)) < 0 and b"bad sizes" in _error()
    assert L.mace_b200_orthogonalize_workspace(2, 300, 400, N.byref(n)) == 0 and n.value > 2 * 300 * 400 * 8
    big = n.value
    assert L.mace_b200_orthogonalize_workspace(4, 300, 400, N.byref(n)) == 0 and n.value > 1.9 * big
    assert L.mace_b200_orthogonalize_workspace(4, 64, 400, N.byref(n)) == 0 and n.value == 0     # stays on the chip
    coef = (ctypes.c_double * 6)(3.4445, -4.7750, 2.0315, 3.4445, -4.7750, 2.0315)
    c = ctypes.addressof(coef)
    orth = lambda steps=2, eps=1e-7, dt=0, ld=4, cp=c: L.mace_b200_orthogonalize(p, 16, ld, p, p, 0, 4, 4, cp, steps, eps, dt, None)  # noqa: E731
    assert orth() == 0
    for kw in (dict(steps=0), dict(steps=17), dict(eps=0.0), dict(eps=float("nan")), dict(dt=3), dict(ld=3), dict(cp=None)):
        assert orth(**kw) < 0 and b"bad arguments" in _error(), kw
    coef[0] = 9.0
    assert orth() < 0 and b"reaches" in _error()


def test_modules_check_arguments():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="activation"):
        X.group_norm(x, 2, activation="elu")
    with pytest.raises(ValueError, match="type of x"):
        X.int8_linear(x, None, None, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        X.int8_linear(torch.zeros(2, 8, dtype=torch.int8), None, None, xscale=x, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="steps"):
        optim.orthogonalize(x, steps=17)
    with pytest.raises(ValueError, match="triple"):
        optim.orthogonalize(x, steps=3, coefficients=((1.0, 0.0, 0.0),) * 2)
    with pytest.raises(ValueError, match="out of range"):
        optim.Muon([torch.nn.Parameter(x)], momentum=1.0)
    with pytest.raises(ValueError, match="matrices"):
        optim.Muon([torch.nn.Parameter(x), torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError, match="optimizer"):
        experts.train_readout(optimizer="sgd")


def test_shape_functions():
    ops = N.ops()
    with FakeTensorMode():
        x = torch.empty(4, 6, 16, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(16, device="cuda")
        assert ops.group_norm(x, 4, w, None, 1e-5, 1, None).shape == x.shape
        y, mean, rstd = ops.group_norm_fwd(x, 4, w, None, 1e-5, 1, None)
        assert mean.shape == rstd.shape == (4, 4) and mean.dtype == torch.float32
        dx, dw, db = ops.group_norm_bwd(y, x, 4, w, None, 1, None, mean, rstd, True, True, False)
        assert dx.shape == x.shape and dw.shape == (16,) and dw.dtype == torch.float32
        off = torch.empty(8, device="cuda", dtype=torch.int64)
        assert ops.group_norm_fwd(x[0], 4, None, None, 1e-5, 0, off)[1].shape == (7, 4)
        q, s = ops.quantize_rows(torch.empty(5, 30, device="cuda"))
        assert q.shape == (5, 30) and q.dtype == torch.int8 and q.stride(0) == 32 and s.shape == (5,)
        y = ops.int8_linear(torch.empty(3, 5, 30, device="cuda"), None, q, s, None, 0)
        assert y.shape == (3, 5, 5) and y.dtype == torch.float32
        assert ops.int8_linear(q, s, q, s, None, 2).dtype == torch.float16
        u = ops.orthogonalize(torch.empty(2, 5, 7, device="cuda"), torch.empty(5, 3, dtype=torch.float64), 1e-7)
        assert u.shape == (2, 5, 7) and u.dtype == torch.bfloat16


CALLS = {
    "group_norm x": lambda o, d: o.group_norm(d(2, 3, 16), 4, None, None, 1e-5, 0, None),
    "group_norm weight": lambda o, d: o.group_norm(torch.empty(2, 3, 16, device="cuda"), 4, d(16), None, 1e-5, 0, None),
    "quantize_rows x": lambda o, d: o.quantize_rows(d(3, 16)),
    "int8_linear x": lambda o, d: o.int8_linear(d(3, 16), None, torch.empty(4, 16, device="cuda", dtype=torch.int8),
                                                torch.empty(4, device="cuda"), None, 0),
    "orthogonalize g": lambda o, d: o.orthogonalize(d(3, 16), torch.empty(5, 3, dtype=torch.float64), 1e-7),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_dual_tensors_are_refused(name):
    ops = N.ops()
    with FakeTensorMode(), fw.dual_level():
        def dual(*shape):
            return fw.make_dual(torch.empty(*shape, device="cuda"), torch.empty(*shape, device="cuda"))

        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[name](ops, dual)


def test_gradients_are_refused_where_there_are_none():
    ops = N.ops()
    with FakeTensorMode():
        x = torch.empty(3, 16, device="cuda", requires_grad=True)
        wq, ws = torch.empty(4, 16, device="cuda", dtype=torch.int8), torch.empty(4, device="cuda")
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.quantize_rows(x)
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.int8_linear(x, None, wq, ws, None, 0)
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.orthogonalize(x, torch.empty(5, 3, dtype=torch.float64), 1e-7)
        with torch.no_grad():
            assert ops.int8_linear(x, None, wq, ws, None, 0).shape == (3, 4)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
def test_plain_group_norm_is_torchs(act):
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 12, 10), (12,), (12,), (3, 12, 10)))
    ins = [t.requires_grad_() for t in (x, w, b)]                # [samples, channels, positions]
    y = torch.nn.functional.group_norm(x, 4, w, b, 1e-5)
    if act:
        y = getattr(torch.nn.functional, act)(y)
    dx, dw, db = torch.autograd.grad(y, ins, dy)
    rows = lambda t: t.detach().transpose(1, 2).reshape(30, 12)  # noqa: E731
    got = R.group_norm_grads(rows(x), 4, w, b, 1e-5, act, [0, 10, 20, 30], rows(dy))
    for a, c in zip(got, (rows(y), rows(dx), dw, db)):
        assert (a - c).abs().max() < 1e-12


def test_rows_of_no_sample_are_zero_in_the_plain_form():
    x = torch.randn(9, 4, dtype=torch.float64)
    one, zero = torch.ones(4, dtype=torch.float64), torch.zeros(4, dtype=torch.float64)
    y = R.group_norm(x, 2, one, zero, 1e-5, None, [2, 2, 5, 5, 8])
    assert not y[:2].any() and not y[8:].any()
    assert torch.equal(y[2:5], R.group_norm(x[2:5], 2, one, zero, 1e-5, None, [0, 3]))
