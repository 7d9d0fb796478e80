"""Dense readouts over per-atom features: group norm with an activation, and linear maps in 8-bit integers to serve them.

    z = group_norm(x, 8, gamma, beta, activation="silu", offsets=offsets)   # over the atoms of each structure
    wq, ws = quantize_rows(w)                                               # once: 8 bits and a scale per output channel
    y = int8_linear(z, wq, ws, bias)                                        # [rows, out], a scale per row of z on the way

They run in sm_100a kernels behind torch.ops.mace_b200.* (float32, bfloat16, float16), on torch's current stream.
`ReadoutBlock` puts them together; `python -m mace_onegpu.readout` trains one over the layer-1 features of a water box with
orthogonalised updates (optim.Muon) and serves it in 8 bits.
"""
from __future__ import annotations

import torch

from .experts import _op

__all__ = ["group_norm", "quantize_rows", "int8_linear", "ReadoutBlock", "Int8Readout"]

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3}


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, activation=None, offsets=None):
    """activation((x - mean) / sqrt(var + eps) * weight + bias), channels last; the statistics are over the positions of a
    sample and the C / groups channels of a group.

    x: [N, .., C], N samples; or [rows, C] with offsets [N + 1] (int32 or int64 on the device, ascending within [0, rows]):
    sample i is rows offsets[i] to offsets[i + 1], rows of no sample give zeros (and get none).  float32, bfloat16 or float16;
    rows may be strided.  weight / bias: [C] of the type of x or float32, or None.  activation: None, "silu", "gelu" (z Phi(z))
    or "relu".  Statistics and parameter gradients are accumulated in fp32, in a fixed order.  Samples are dealt out by
    their mean length: one a thousand times as long as the others is right, but slow.  Differentiable once.  A sample whose offsets
    leave the rows is NaN; where they descend anywhere, all rows are."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu', 'gelu' or 'relu' (got {activation!r})")
    return _op("group_norm")(x, int(groups), weight, bias, float(eps), ACTIVATIONS[activation], offsets)


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def quantize_rows(x):
    """Rows of x [.., K] in 8 bits: (q int8 [.., K], scale float32 [..]) with scale = max |row| / 127 and q the nearest whole
    numbers of row / scale (of the exact quotient, ties to even).  q's rows lie whole 16 bytes apart, as int8_linear reads them.
    A row with NaN or an infinity has that scale.  No gradient."""
    return _op("quantize_rows")(x)


def int8_linear(x, wq, wscale, bias=None, *, xscale=None, out_dtype=None):
    """x [.., K] times wq [N, K] (int8) in 8-bit integers: y [.., N] = (q . wq) scale wscale + bias.

    x: float32, bfloat16 or float16, quantized by row on the way, the result has its type; or int8 with xscale [..] (float32),
    the result has out_dtype (float32 by default).  wscale: float32 [N]; wq, wscale = quantize_rows(w).  bias: [N] of the result's
    type or float32.  Sums are exact (K at most 131,071), y is rounded once.  Rows of 8-bit values that do not lie whole 16
    bytes apart are copied first.  No gradient."""
    if x.dtype != torch.int8:
        if out_dtype is not None and out_dtype != x.dtype:
            raise ValueError(f"the result has the type of x (out_dtype {out_dtype}, x {x.dtype})")
        out_dtype = x.dtype
    elif out_dtype is None:
        out_dtype = torch.float32
    if out_dtype not in _TYPES:
        raise ValueError(f"x / out_dtype must be float32, bfloat16 or float16 (got {out_dtype})")
    return _op("int8_linear")(x, xscale, wq, wscale, bias, _TYPES[out_dtype])


class ReadoutBlock(torch.nn.Module):
    """Two linear maps, each after a group norm with silu over the atoms of a structure: out = W2 f(norm(W1 f(norm(x)) + b1)) + b2.

    x [rows, dim] (rows may be strided) -> [rows, out]; offsets as in group_norm, None: all rows are one structure."""

    def __init__(self, dim, hidden, out, groups, dtype=torch.float32, device="cuda", seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)

        def par(*shape, scale=0.0, mean=0.0):
            return torch.nn.Parameter((torch.randn(*shape, generator=g) * scale + mean).to(device=device, dtype=dtype))

        self.groups = int(groups)
        self.gamma1, self.beta1 = par(dim, mean=1.0), par(dim)
        self.w1, self.b1 = par(hidden, dim, scale=dim ** -0.5), par(hidden)
        self.gamma2, self.beta2 = par(hidden, mean=1.0), par(hidden)
        self.w2, self.b2 = par(out, hidden, scale=hidden ** -0.5), par(out)

    def _norm(self, x, gamma, beta, offsets):
        if offsets is not None:
            return group_norm(x, self.groups, gamma, beta, activation="silu", offsets=offsets)
        return group_norm(x[None], self.groups, gamma, beta, activation="silu")[0]

    def forward(self, x, offsets=None):
        h = torch.nn.functional.linear(self._norm(x, self.gamma1, self.beta1, offsets), self.w1, self.b1)
        return torch.nn.functional.linear(self._norm(h, self.gamma2, self.beta2, offsets), self.w2, self.b2)

    def matrices(self):
        """What optim.Muon takes; the other parameters are vectors."""
        return [self.w1, self.w2]

    def vectors(self):
        return [p for p in self.parameters() if p.dim() < 2]

    def quantized(self):
        """An Int8Readout of the block as it is now."""
        return Int8Readout(self)


def _rows16(q):
    """8-bit rows that lie whole 16 bytes apart: q itself, or a copy."""
    if (q.shape[1] == 1 or q.stride(1) == 1) and q.stride(0) % 16 == 0 and q.stride(0) >= q.shape[1]:
        return q
    return q.new_zeros(q.shape[0], (q.shape[1] + 15) // 16 * 16)[:, :q.shape[1]].copy_(q)


class Int8Readout(torch.nn.Module):
    """A ReadoutBlock with its matrices in 8 bits and a scale per output channel; a scale per row of the activations is taken on the
    way.  For inference: no gradient.  Casts of the module (.half(), .to(torch.bfloat16)) are casts of the norms and biases: the scales
    stay float32, and rows of the matrices whole 16 bytes apart wherever the module is moved."""

    def __init__(self, block):
        super().__init__()
        self.groups = block.groups
        with torch.no_grad():
            for name in ("gamma1", "beta1", "b1", "gamma2", "beta2", "b2"):
                self.register_buffer(name, getattr(block, name).detach().clone())
            for i, w in ((1, block.w1), (2, block.w2)):
                q, s = quantize_rows(w.detach())
                self.register_buffer(f"wq{i}", q)
                self.register_buffer(f"ws{i}", s)

    _norm = ReadoutBlock._norm

    def _apply(self, fn, recurse=True):
        scales = {name: self._buffers[name] for name in ("ws1", "ws2")}
        super()._apply(fn, recurse)
        for name, kept in scales.items():
            if self._buffers[name].dtype != torch.float32:
                self._buffers[name] = kept.to(self._buffers[name].device)
        for name in ("wq1", "wq2"):
            self._buffers[name] = _rows16(self._buffers[name])
        return self

    @torch.no_grad()
    def forward(self, x, offsets=None):
        h = int8_linear(self._norm(x, self.gamma1, self.beta1, offsets), self.wq1, self.ws1, self.b1)
        return int8_linear(self._norm(h, self.gamma2, self.beta2, offsets), self.wq2, self.ws2, self.b2)


def train_readout(n=8, hidden=256, groups=8, steps=200, lr=0.02, lr_vectors=3e-3, dtype=torch.float32, seed=0):
    """Trains a ReadoutBlock to give the per-atom energies of the model from its layer-1 scalar features H1[:, 0e] of a water
    box of 3 n^3 atoms (random-init weights), the matrices with Muon, the vectors with Adam; then serves it in 8 bits.
    Returns a dict of what happened."""
    import time

    from . import experts, optim

    x, target = experts.water_features(n, dtype, seed)
    block = ReadoutBlock(x.shape[1], hidden, 1, groups, dtype=dtype, seed=seed)
    opts = [optim.Muon(block.matrices(), lr=lr), torch.optim.Adam(block.vectors(), lr=lr_vectors)]
    losses = []
    t0 = time.perf_counter()
    for _ in range(steps):
        for opt in opts:
            opt.zero_grad()
        loss = torch.nn.functional.mse_loss(block(x).float(), target.float())
        loss.backward()
        for opt in opts:
            opt.step()
        losses.append(loss.detach())
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    with torch.no_grad():
        y, y8 = block(x).float(), block.quantized()(x).float()
    return {"atoms": len(x), "hidden": hidden, "groups": groups, "steps": steps, "dtype": str(dtype).split(".")[-1],
            "loss_first": float(losses[0]), "loss_last": float(losses[-1]), "steps_per_s": steps / dt,
            "int8_loss": float(torch.nn.functional.mse_loss(y8, target.float())),
            "int8_rel": float((y8 - y).norm() / y.norm())}


def main():
    import argparse
    import json

    ap = argparse.ArgumentParser(description="Train a dense readout over layer-1 features of a water box and serve it in 8 bits")
    ap.add_argument("--n", type=int, default=8, help="molecules along an edge (3 n^3 atoms)")
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--groups", type=int, default=8)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--lr", type=float, default=0.02, help="of the matrices (Muon)")
    ap.add_argument("--lr-vectors", type=float, default=3e-3, help="of norms and biases (Adam)")
    ap.add_argument("--dtype", default="float32", choices=["float32", "bfloat16", "float16"])
    a = ap.parse_args()
    print(json.dumps(train_readout(a.n, a.hidden, a.groups, a.steps, a.lr, a.lr_vectors, getattr(torch, a.dtype))))


if __name__ == "__main__":
    main()
