"""Mixtures of linear experts over per-atom features: layer norm, routing, and products with per-atom matrices.

The species skip of the interaction blocks (mace_onegpu/fast_layers.py:96-105 in the reference) sends every atom through
the matrix of its species.  Here the matrix is chosen by a trained router, several per atom if wanted:

    xn = layer_norm(x, gamma, beta)                        # [T, D], rows may be strided: h1[:, 0] of [T, 4, 128]
    weights, experts = route(xn @ wr.T, k)                 # [T, k] each
    y = expert_linear(xn, w, plan_experts(experts, E), weights)   # sum_j weights[t, j] w[experts[t, j]] xn[t]

All three run in sm_100a kernels behind torch.ops.mace_b200.* (float32, bfloat16, float16), on torch's current stream,
and are differentiable (once).  `ExpertBlock` puts them together; `python -m mace_onegpu.experts` trains one as a readout
over the layer-1 features of a water box.
"""
from __future__ import annotations

import torch

from . import _native as N

__all__ = ["layer_norm", "route", "ExpertPlan", "plan_experts", "expert_linear", "ExpertBlock"]

# Forward calls that need no gradient read their matrices once per slot, without sorting the slots by expert, while that is
# at most FEW_BYTES and FEW_SLOTS slots.  B200, per-slot form against plan + tensor cores: 34 MB (4 tokens, k 4, 1024 x 1024
# bf16) 9.7 / 27.7 us, 65 MB (500, 2, 128 x 128 fp32) 14.3 / 19.1, 134 MB (16, 1, 2048 x 2048 bf16) 31 / 23, 157 MB (600, 2,
# 256 x 256 bf16) 31 / 24.
FEW_BYTES = 96 << 20
FEW_SLOTS = 4096


_OPS = {}


def _op(name):
    """The op's only overload (looked up once: resolving it again costs a small call a microsecond)."""
    if name not in _OPS:
        _OPS[name] = getattr(N.ops(), name).default
    return _OPS[name]


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [.., D].

    x: float32, bfloat16 or float16; its rows may be strided.  weight / bias: [D] of the type of x or float32, or None.
    Statistics and parameter gradients are accumulated in fp32, in a fixed order."""
    return _op("layer_norm")(x, weight, bias, float(eps))


def route(logits, k, *, bias=None, score="softmax", groups=1, top_groups=1, renormalize=True, scale=1.0):
    """Chooses k of E experts per row of logits [T, E].  Returns (weights [T, k] float32, experts [T, k] int32), best
    first.

    score: "softmax" or "sigmoid" of the logits.  The choice ranks by score + bias (bias: float32 [E], for balance; it
    does not enter the weights and gets no gradient), by the logits when bias is None; ties go to the lowest index.
    Logits of -inf are closed: where fewer than k experts are open the remaining slots get expert -1 and weight 0.
    groups > 1: the E experts are `groups` runs of E / groups, and only the top_groups runs with the highest sum of
    their two best values stay open.  weights: scores, divided by the sum over the chosen ones if `renormalize`, times
    `scale`.  Differentiable w.r.t. the logits."""
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"score must be 'softmax' or 'sigmoid' (got {score!r})")
    return _op("route")(logits, bias, int(k), score == "softmax", int(groups), int(top_groups), bool(renormalize),
                        float(scale))


class ExpertPlan:
    """The slots (token, choice) of `experts` [T, k] (or [T]) in expert order, for any number of expert_linear calls
    with the same choice.  An expert of -1 means none.  Sorted on the device at the first product that needs it."""

    def __init__(self, experts, n_experts):
        if experts.dim() not in (1, 2) or experts.dtype not in (torch.int32, torch.int64):
            raise ValueError("experts must be an integer tensor [tokens, k] or [tokens]")
        if not 1 <= int(n_experts):
            raise ValueError("n_experts must be positive")
        self.experts = (experts if experts.dim() == 2 else experts[:, None]).to(torch.int32).contiguous()
        self.n_experts = int(n_experts)
        self._words = None

    @property
    def words(self):
        """The plan as the kernels read it (int32)."""
        if self._words is None:
            self._words = _op("expert_plan")(self.experts, self.n_experts)
        return self._words

    def check(self):
        """Reads the device status word (synchronises) and raises if an index was outside [-1, n_experts) or a product
        gave up waiting."""
        st = int(self.words[1].item())
        if st & N.ST_BAD_EXPERT:
            raise RuntimeError(f"expert index outside [-1, {self.n_experts})")
        if st & N.ST_TC_TIMEOUT:
            raise RuntimeError("expert_linear: a tensor-core kernel gave up waiting; its outputs are not valid")


def plan_experts(experts, n_experts):
    """ExpertPlan(experts, n_experts)."""
    return ExpertPlan(experts, n_experts)


def expert_linear(x, w, plan, weights=None):
    """Products with the matrices w [E, O, D] that the plan assigns.

    x: [T, D], or [T, k, D] with a row per slot.  weights [T, k] float32: out [T, O] = sum_j weights[t, j] w[e_tj] x;
    None: out [T, k, O] = w[e_tj] x.  x and w: float32 (at fp32 accuracy), bfloat16 or float16.  Slots with expert -1
    give zeros and no gradient.  Differentiable w.r.t. x, w and weights; sums run in a fixed order."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError("plan must be an ExpertPlan (plan_experts(experts, n_experts))")
    if w.dim() != 3 or w.shape[0] != plan.n_experts:
        raise ValueError(f"w must be [{plan.n_experts}, out, in] (got {tuple(w.shape)})")
    grad = torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or
                                        (weights is not None and weights.requires_grad))
    slots = plan.experts.numel()
    few = not grad and slots <= FEW_SLOTS and slots * w[0].numel() * w.element_size() <= FEW_BYTES
    return _op("expert_linear")(x, w, plan.experts, None if few else plan.words, weights)
