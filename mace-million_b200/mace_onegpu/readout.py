"""Dense readouts over per-atom features: group norm with an activation, and linear maps in 8-bit integers to serve them.

    z = group_norm(x, 8, gamma, beta, activation="silu", offsets=offsets)   # over the atoms of each structure
    wq, ws = quantize_rows(w)                                               # once: 8 bits and a scale per output channel
    y = int8_linear(z, wq, ws, bias)                                        # [rows, out], a scale per row of z on the way

They run in sm_100a kernels behind torch.ops.mace_b200.* (float32, bfloat16, float16), on torch's current stream.
"""
from __future__ import annotations

import torch

from .experts import _op

__all__ = ["group_norm", "quantize_rows", "int8_linear"]

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3}


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, activation=None, offsets=None):
    """activation((x - mean) / sqrt(var + eps) * weight + bias), channels last; the statistics are over the positions of a
    sample and the C / groups channels of a group.

    x: [N, .., C], N samples; or [rows, C] with offsets [N + 1] (int32 or int64 on the device, ascending within [0, rows]):
    sample i is rows offsets[i] to offsets[i + 1], rows of no sample give zeros (and get none).  float32, bfloat16 or float16;
    rows may be strided.  weight / bias: [C] of the type of x or float32, or None.  activation: None, "silu", "gelu" (z Phi(z))
    or "relu".  Statistics and parameter gradients are accumulated in fp32, in a fixed order.  Differentiable once.  A sample
    whose offsets descend or leave the rows is NaN."""
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
