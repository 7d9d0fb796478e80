"""Plain fp64 forms of the readout operators (tests only)."""
import math

import torch


def activation(z, name):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    return torch.where(z < 0, torch.zeros_like(z), z) if name == "relu" else z


def group_norm(x, groups, w, b, eps, act, edges):
    """x [rows, C] in fp64; edges: first row of each sample and the end of the last.  Rows of no sample are zero."""
    c = x.shape[1]
    parts, at = [], 0
    for lo, hi in zip(edges, edges[1:]):
        if lo > at:
            parts.append(x[at:lo] * 0)
        at = hi
        if hi == lo:
            continue
        v = x[lo:hi].reshape(hi - lo, groups, c // groups)
        mu = v.mean((0, 2), keepdim=True)
        var = ((v - mu) ** 2).mean((0, 2), keepdim=True)
        z = ((v - mu) / torch.sqrt(var + eps)).reshape(hi - lo, c)
        parts.append(activation(z * w + b, act))
    if at < x.shape[0]:
        parts.append(x[at:] * 0)
    return torch.cat(parts) if parts else x * 0


def group_norm_grads(x, groups, w, b, eps, act, edges, dy):
    ins = [t.detach().double().requires_grad_() for t in (x, w, b)]
    y = group_norm(ins[0], groups, ins[1], ins[2], eps, act, edges)
    return (y.detach(), *torch.autograd.grad(y, ins, dy.double()))
