"""Dense readouts over per-atom features: group norm with an activation.

    z = group_norm(x, 8, gamma, beta, activation="silu", offsets=offsets)   # over the atoms of each structure

It runs in sm_100a kernels behind torch.ops.mace_b200.* (float32, bfloat16, float16), on torch's current stream.
"""
from __future__ import annotations

from .experts import _op

__all__ = ["group_norm"]

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
