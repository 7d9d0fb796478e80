"""Products in 8-bit integers (mace_onegpu.readout.quantize_rows, int8_linear) against the plain form in 64 bits: whole numbers have
to be equal (ties, tiny and huge rows, zero rows), results are one fp32 expression of an exact sum.

Tolerances.  y = fma(float(sum) s, w, b): three roundings of fp32 relative to |sum s w| and |b| (2^-22 of them), then one rounding
to the type: 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32)."""
import pytest
import torch

from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _quantize(x):
    """The definition: the scale is an fp32 number, the quotient is exact to 53 bits (ties are exact in it)."""
    top = x.float().abs().amax(-1)
    scale = (top.double() / 127).float()
    q = torch.round(x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[..., None])
    return torch.where(scale[..., None] > 0, q, torch.zeros_like(q)), scale


def _close(y, q, s, wq, ws, b, dt):
    part = (q.double() @ wq.double().T) * (s.double()[:, None] * ws.double())
    want = part if b is None else part + b.double()
    tol = U[dt] * want.abs() + 2.0 ** -22 * (part.abs() + (0 if b is None else b.double().abs())) + (2.0 ** -25 if dt == torch.float16 else 0)
    assert y.dtype == dt and y.shape == want.shape
    bad = ~((y.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((y.double() - want).abs().max())}"


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 16), (100, 128), (33, 515), (9, 4096), (2, 5000), (70000, 24)])
def test_quantize_rows(rows, k, dt):
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=g, device="cuda") * 3).to(DT[dt])
    x[rows // 2] = 0
    q, s = X.quantize_rows(x)
    q0, s0 = _quantize(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and (rows == 1 or q.stride(0) % 16 == 0)
    assert torch.equal(s, s0) and torch.equal(q.double(), q0)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k", [(2500, 256), (37, 504), (9, 1016), (2501, 1032), (300, 2048), (5, 2064), (601, 4112), (7, 8192), (601, 8208),
                                    (3, 16384), (3, 16400)])
def test_quantize_rows_of_each_width(rows, k, dt):
    """Whole vectors on either side of the widths that a warp, half a block and a block hold; some rows of whole numbers, full of ties."""
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[1::3] = torch.randint(-254, 255, x[1::3].shape, generator=g, device="cuda").float() / 2
    x[1::3, k // 2] = 127
    x = x.to(DT[dt])
    q, s = X.quantize_rows(x)
    q0, s0 = _quantize(x)
    assert torch.equal(s, s0) and torch.equal(q.double(), q0)


@pytest.mark.parametrize("n", [3551, 3552, 3557, 4735, 4736, 4739])
def test_few_tokens_and_many_channels(n):
    """One, two and four rows of the weights a warp, the last ones incomplete."""
    g = torch.Generator(device="cuda").manual_seed(n)
    wq, ws = X.quantize_rows(torch.randn(n, 200, generator=g, device="cuda"))
    for tokens in (1, 2, 3, 4):
        x = torch.randn(tokens, 200, generator=g, device="cuda", dtype=torch.bfloat16)
        q, s = _quantize(x)
        b = torch.randn(n, generator=g, device="cuda")
        _close(X.int8_linear(x, wq, ws, b), q, s, wq, ws, b, torch.bfloat16)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("k,ld", [(4, 4), (7, 9), (8, 11), (15, 15), (17, 40), (131, 131), (260, 263), (515, 515), (771, 772), (1023, 1025),
                                  (4099, 4099), (8193, 8200), (17001, 17001)])
def test_quantize_rows_of_any_alignment(k, ld, dt):
    """Rows that start anywhere, up to the first and the last element of their storage; what lies between them is NaN."""
    g = torch.Generator(device="cuda").manual_seed(k)
    for first in (0, 1, 5):
        rows = 9
        store = torch.full((first + (rows - 1) * ld + k,), float("nan"), device="cuda", dtype=DT[dt])
        x = store.as_strided((rows, k), (ld, 1), first)
        x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
        q, s = X.quantize_rows(x)
        q0, s0 = _quantize(x)
        assert torch.equal(s, s0) and torch.equal(q.double(), q0)
        pad = q.as_strided((rows, q.stride(0) - k), (q.stride(0), 1), q.storage_offset() + k)
        assert not pad[:-1].any()


def test_quantize_ties_and_extremes():
    """Rows whose largest value is 127 times a power of two have exact ties at every half; scales down to subnormal ones."""
    half = torch.arange(-254, 255, device="cuda").float() / 2
    rows = torch.stack([half * 2.0 ** e for e in (0, -100, 100, 1, -126, -140, -148)])
    q, s = X.quantize_rows(rows)
    q0, s0 = _quantize(rows)
    assert torch.equal(s, s0) and torch.equal(q.double(), q0.clamp(-127, 127))
    rows = torch.randn(400, 1000, device="cuda") * torch.logspace(-44, 37, 400, device="cuda")[:, None]
    q, s = X.quantize_rows(rows)
    q0, s0 = _quantize(rows)
    assert torch.equal(s, s0) and torch.equal(q.double(), q0.clamp(-127, 127))
    bad = torch.randn(3, 64, device="cuda")
    bad[0, 5], bad[1, 6] = float("nan"), float("-inf")
    q, s = X.quantize_rows(bad)
    assert s[0].isnan() and s[1].isinf() and not q[:2].any() and q[2].any()
    w = torch.randint(-127, 128, (20, 64), dtype=torch.int8, device="cuda")
    for rep in (1, 20):                                       # both kernels
        y = X.int8_linear(bad.repeat(rep, 1), w, torch.ones(20, device="cuda")).view(rep, 3, 20)
        assert y[:, :2].isnan().all() and y[:, 2].isfinite().all()


SIZES = [(1, 1, 1), (1, 1024, 1024), (1, 515, 1001), (2, 128, 512), (3, 33, 7), (4, 4096, 300), (5, 1000, 999), (8, 2048, 5000),
         (8, 20000, 40), (9, 16, 8), (17, 128, 512), (64, 515, 130), (192, 128, 512), (300, 1000, 257), (1000, 2048, 1024),
         (4097, 640, 777), (20000, 64, 64), (6000, 1024, 4096), (37, 131071, 33), (1, 131071, 9)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,k,n", SIZES)
def test_int8_linear(t, k, n, dt):
    dt = DT[dt]
    g = torch.Generator(device="cuda").manual_seed(t + k + n)
    x = (torch.randn(t, k, generator=g, device="cuda") * 2).to(dt)
    wq, ws = X.quantize_rows(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    b = torch.randn(n, generator=g, device="cuda").to(dt) if t % 2 else None
    q, s = _quantize(x)
    y = X.int8_linear(x, wq, ws, b)
    _close(y, q, s, wq, ws, b, dt)
    got, sg = X.quantize_rows(x)
    assert torch.equal(X.int8_linear(got, wq, ws, b, xscale=sg, out_dtype=dt), y)


@pytest.mark.parametrize("t", [1, 7, 40, 500])
def test_whole_range_of_values(t):
    """-128 and 127 at the longest sums: the sums need all of int32."""
    k = 131071
    q = torch.full((t, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    y = X.int8_linear(q, w, torch.ones(3, device="cuda"), xscale=torch.ones(t, device="cuda"))
    assert (y == torch.tensor([128.0 * 128 * k, -128.0 * 127 * k, 128.0 * 128 * k], device="cuda").float()).all()


def test_strides_shapes_and_types():
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(50, 4, 128, generator=g, device="cuda")
    wq, ws = X.quantize_rows(torch.randn(40, 128, generator=g, device="cuda"))
    y = X.int8_linear(h[:, 0], wq, ws)
    assert torch.equal(y, X.int8_linear(h[:, 0].contiguous(), wq, ws))
    assert torch.equal(X.int8_linear(h, wq, ws)[:, 0], y) and X.int8_linear(h, wq, ws).shape == (50, 4, 40)
    assert torch.equal(X.int8_linear(h[3, 0], wq, ws), y[3])
    odd = torch.randn(50, 131, generator=g, device="cuda")[:, 3:]          # rows that start off any vector
    assert torch.equal(X.int8_linear(odd, wq, ws), X.int8_linear(odd.contiguous(), wq, ws))
    assert torch.equal(X.int8_linear(odd[:5], wq, ws), X.int8_linear(odd, wq, ws)[:5])
    wide = torch.zeros(40, 133, dtype=torch.int8, device="cuda")
    wide[:, 5:] = wq
    assert torch.equal(X.int8_linear(h[:, 0], wide[:, 5:], ws), y)         # rows off 16 bytes: copied
    assert torch.equal(X.int8_linear(h[:, 0], wq.T.contiguous().T, ws), y)
    q, s = X.quantize_rows(h)
    assert q.shape == h.shape and s.shape == (50, 4)
    assert torch.equal(X.int8_linear(q[:, 0], wq, ws, xscale=s[:, 0]), y)
    half = X.int8_linear(h[:, 0].half(), wq, ws, torch.ones(40, device="cuda"))
    assert half.dtype == torch.float16
    assert X.int8_linear(h[:0], wq, ws).shape == (0, 4, 40)


def test_refusals():
    x = torch.randn(4, 32, device="cuda")
    wq, ws = X.quantize_rows(torch.randn(8, 32, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradient"):
        X.int8_linear(x.clone().requires_grad_(), wq, ws)
    with pytest.raises(RuntimeError, match="no gradient"):
        X.quantize_rows(x.clone().requires_grad_())
    with torch.no_grad():
        X.int8_linear(x.clone().requires_grad_(), wq, ws)
    with pytest.raises(RuntimeError, match="int8"):
        X.int8_linear(x, wq.float(), ws)
    with pytest.raises(RuntimeError, match="x must be"):
        X.int8_linear(x[:, :31], wq, ws)
    with pytest.raises(RuntimeError, match="wscale"):
        X.int8_linear(x, wq, ws[:7])
    with pytest.raises(RuntimeError, match="bias"):
        X.int8_linear(x, wq, ws, torch.ones(8, device="cuda").half())
    with pytest.raises(RuntimeError, match="needs xscale"):
        X.int8_linear(wq, wq, ws)
    with pytest.raises(RuntimeError, match="goes with 8-bit"):
        X.int8_linear(x, wq, ws, xscale=ws)
    with pytest.raises(RuntimeError, match="a value for each token"):
        X.int8_linear(wq, wq, ws, xscale=ws[:3])
    with pytest.raises(ValueError, match="type of x"):
        X.int8_linear(x, wq, ws, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        X.int8_linear(x.double(), wq, ws)
    with pytest.raises(RuntimeError, match="columns"):
        X.int8_linear(torch.zeros(1, 131072, device="cuda"), torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), ws[:1])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        X.int8_linear(x, wq.cpu(), ws)


def test_streams_and_graphs():
    x = torch.randn(600, 128, device="cuda")
    wq, ws = X.quantize_rows(torch.randn(64, 128, device="cuda"))
    want, one = X.int8_linear(x, wq, ws), X.int8_linear(x[:1], wq, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = X.int8_linear(x, wq, ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            held, held1 = X.int8_linear(x, wq, ws), X.int8_linear(x[:1], wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want) and torch.equal(held1, one)
    x.neg_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, -want) and torch.equal(held1, -one)
