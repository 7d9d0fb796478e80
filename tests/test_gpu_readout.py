"""The readout operators as they are used together: a ReadoutBlock over ragged structures whose gradients are compared with fp64
autograd of the same formulas, Muon steps with it, its 8-bit form, and the two training commands.

Tolerances.  float32 parts: sums of up to 128 products, norms over up to 1000 values and their chain through two layers come to
within 1e-4 of the largest gradient (each product of matrices is torch's, in fp32 with 10-bit TF32 switched off).  8 bits: a value is
off by at most half a step, scale / 2 = max / 254; with independent roundings a sum of K products is off by its root mean square
factor 2^0.5 / 254 max / rms / 3^0.5, about 1.3% for max / rms of 4, twice (two layers)."""
import json
import os
import subprocess
import sys

import pytest
import torch

import readout_refs as R
from mace_onegpu import optim
from mace_onegpu import readout as X

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _plain(p, groups, x, edges):
    h = R.group_norm(x, groups, p["gamma1"], p["beta1"], 1e-5, "silu", edges) @ p["w1"].T + p["b1"]
    return R.group_norm(h, groups, p["gamma2"], p["beta2"], 1e-5, "silu", edges) @ p["w2"].T + p["b2"]


def _block(seed=3):
    block = X.ReadoutBlock(48, 64, 5, 4, seed=seed)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in block.vectors():
            p += 0.2 * torch.randn(p.shape, generator=g).cuda()
    return block


EDGES = [0, 1, 1, 90, 250, 333]


def test_gradients_through_the_block():
    block, g = _block(), torch.Generator().manual_seed(0)
    x, dy = torch.randn(333, 4, 48, generator=g), torch.randn(333, 5, generator=g)
    off = torch.tensor(EDGES).cuda()
    xd = x.cuda().requires_grad_()
    y = block(xd[:, 0], off)
    names = [n for n, _ in block.named_parameters()]
    got = torch.autograd.grad(y, [xd, *block.parameters()], dy.cuda())
    p = {n: v.detach().cpu().double().requires_grad_() for n, v in block.named_parameters()}
    x0 = x[:, 0].double().requires_grad_()
    want = _plain(p, 4, x0, EDGES)
    assert (y.detach().cpu() - want).abs().max() < 1e-4 * want.abs().max()
    grads = torch.autograd.grad(want, [x0, *(p[n] for n in names)], dy.double())
    assert (got[0][:, 0].cpu() - grads[0]).abs().max() < 1e-4 * grads[0].abs().max() and not got[0][:, 1:].any()
    for n, a, b in zip(names, got[1:], grads[1:]):
        assert (a.cpu() - b).abs().max() < 1e-4 * b.abs().max(), n


def test_one_structure_without_offsets():
    block = _block()
    x = torch.randn(120, 48, device="cuda")
    assert torch.allclose(block(x), block(x, torch.tensor([0, 120]).cuda()), atol=1e-5)


def test_training_steps_and_serving():
    """Muon and Adam steps leave finite parameters that a graph replay repeats; the 8-bit form follows the block."""
    block, g = _block(), torch.Generator(device="cuda").manual_seed(1)
    x, target = torch.randn(333, 48, device="cuda", generator=g), torch.randn(333, 5, device="cuda", generator=g)
    off = torch.tensor(EDGES).cuda()
    opts = [optim.Muon(block.matrices(), lr=0.02), torch.optim.Adam(block.vectors(), lr=1e-3)]
    before = block.w1.detach().clone()
    for _ in range(3):
        loss = torch.nn.functional.mse_loss(block(x, off), target)
        for o in opts:
            o.zero_grad()
        loss.backward()
        for o in opts:
            o.step()
    # an update of Muon has singular values of 0.6 to 1.3: 3 steps of lr max(1, 64 / 48)^0.5 move the matrix by at most this
    moved = (block.w1.detach() - before).double()
    assert 0 < float(torch.linalg.matrix_norm(moved, 2)) < 3 * 0.02 * (64 / 48) ** 0.5 * 1.3
    served = block.quantized()
    with torch.no_grad():
        y = block(x, off)
    y8 = served(x, off)
    assert not y8.requires_grad and float((y8 - y).norm() / y.norm()) < 0.05
    # the served block is the formula of the 8-bit products on the same norms
    z = X.group_norm(x, 4, block.gamma1.detach(), block.beta1.detach(), activation="silu", offsets=off)
    h = X.int8_linear(z, *X.quantize_rows(block.w1.detach()), block.b1.detach())
    z = X.group_norm(h, 4, block.gamma2.detach(), block.beta2.detach(), activation="silu", offsets=off)
    assert torch.equal(X.int8_linear(z, *X.quantize_rows(block.w2.detach()), block.b2.detach()), y8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = served(x, off)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, y8)
    again = torch.load(_saved(served), weights_only=False)
    assert torch.equal(again(x, off), y8)


def _saved(module):
    import io

    f = io.BytesIO()
    torch.save(module, f)
    f.seek(0)
    return f


def test_two_graphs_have_workspaces_of_their_own():
    a, b = torch.randn(3, 200, 260, device="cuda"), torch.randn(2, 300, 170, device="cuda")
    x, y = torch.randn(40, 3000, 64, device="cuda"), torch.randn(30, 4000, 64, device="cuda")   # beyond the chip: in two launches
    want = [optim.orthogonalize(a), optim.orthogonalize(b), X.group_norm(x, 8), X.group_norm(y, 8)]
    torch.cuda.synchronize()
    graphs, held = [], []
    for u, v in ((a, x), (b, y)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append((optim.orthogonalize(u), X.group_norm(v, 8)))
        graphs.append(g)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for st, g in zip(s, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0][0], want[0]) and torch.equal(held[1][0], want[1])
    assert torch.equal(held[0][1], want[2]) and torch.equal(held[1][1], want[3])


@pytest.mark.parametrize("b,m,n", [(1, 1100, 1300), (1, 2304, 2304), (150, 90, 200)])
def test_two_calls_at_once(b, m, n):
    """Two grids whose CTAs wait on one another, each as wide as the GPU, on two streams."""
    a, c = torch.randn(b, m, n, device="cuda"), torch.randn(b, m, n, device="cuda")
    want = optim.orthogonalize(a), optim.orthogonalize(c)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, g in zip(s, (a, c)):
            with torch.cuda.stream(st):
                got.append(optim.orthogonalize(g))
    torch.cuda.synchronize()
    for i, u in enumerate(got):
        assert torch.equal(u, want[i % 2])


def test_offsets_beyond_32_bits():
    """Elements past 2^31: the last rows are those of a call of their own."""
    rows, c = 70_000_003, 32
    x = torch.empty(rows, c, device="cuda", dtype=torch.bfloat16).normal_()
    y = X.group_norm(x, 4, activation="silu", offsets=torch.tensor([0, rows - 100, rows]).cuda())
    # a sample in another cut: the same values but for the order of sums, an ulp of bf16 (2^-8 relative) of values up to 5
    assert (y[-100:].float() - X.group_norm(x[None, -100:], 4, activation="silu")[0].float()).abs().max() < 0.04
    head = x[:1000].double().view(1000, 4, 8)
    mean = torch.stack([x[:-100, 8 * g:8 * g + 8].float().mean(0).double().mean() for g in range(4)])
    assert mean.abs().max() < 1e-3                            # of 5.6e8 normal values: 4e-5 and the order of an fp32 sum
    assert (y[:1000].double() - R.activation(head.reshape(1000, c), "silu")).abs().max() < 0.05
    del x, y, head
    t, k, n = 2_200_000, 64, 1000
    x = torch.empty(t, k, device="cuda", dtype=torch.float16).normal_()
    wq, ws = X.quantize_rows(torch.randn(n, k, device="cuda"))
    y = X.int8_linear(x, wq, ws)
    assert torch.equal(y[-50:], X.int8_linear(x[-50:], wq, ws)) and torch.equal(y[-2:], X.int8_linear(x[-2:], wq, ws))
    del x, y
    g = torch.empty(65535, 100, 330, device="cuda", dtype=torch.bfloat16).normal_()
    u = optim.orthogonalize(g)
    assert torch.equal(u[-3:], optim.orthogonalize(g[-3:]))


@pytest.mark.parametrize("args", [["mace_onegpu.readout", "--n", "4", "--steps", "3", "--hidden", "32"],
                                  ["mace_onegpu.readout", "--n", "4", "--steps", "3", "--hidden", "32", "--dtype", "bfloat16"],
                                  ["mace_onegpu.experts", "--n", "4", "--steps", "3", "--optimizer", "muon"],
                                  ["mace_onegpu.experts", "--n", "4", "--steps", "3"]])
def test_commands(args):
    out = subprocess.run([sys.executable, "-m", *args], cwd=os.path.join(ROOT, "mace-million_b200"), capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    d = json.loads(out.stdout.strip().splitlines()[-1])
    assert d["atoms"] == 192 and d["steps"] == 3 and d["loss_first"] == d["loss_first"] and d["loss_last"] == d["loss_last"]
