"""Training of the matrices of a readout: orthogonalised updates, and an optimiser that takes them.

    u = orthogonalize(g)          # [.., m, n] -> bfloat16: singular values of every matrix moved towards one

    opt = Muon([p for p in block.parameters() if p.dim() >= 2], lr=0.02)

`orthogonalize` runs in sm_100a kernels behind torch.ops.mace_b200.*, on torch's current stream.  Expert matrices [E, O, D] are
a batch of E matrices.
"""
from __future__ import annotations

import torch

from . import _native
from .experts import _op

__all__ = ["orthogonalize", "Muon", "COEFFICIENTS"]

# a, b, c of the odd polynomial a s + b s^3 + c s^5: steep at zero, and every s of (0, 1] stays near one after a few steps
COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_TABLES = {}


def _table(steps, coefficients):
    """float64 [steps, 3] in host memory, made once for each argument."""
    key = (steps, tuple(map(tuple, coefficients)) if isinstance(coefficients[0], (tuple, list)) else tuple(coefficients))
    table = _TABLES.get(key)
    if table is None:
        rows = key[1] if isinstance(key[1][0], tuple) else (key[1],) * steps
        if len(rows) != steps or any(len(r) != 3 for r in rows):
            raise ValueError(f"coefficients must be (a, b, c), or one such triple for each of the {steps} steps")
        table = torch.tensor(rows, dtype=torch.float64, device="cpu")
        if type(table) is torch.Tensor:             # (a shape tensor has no values to keep)
            if len(_TABLES) > 64:                   # other threads may have dropped or added tables meanwhile
                _TABLES.clear()
            _TABLES[key] = table
    return table


_TAKEN = set()


def _check_polynomial(steps, coefficients, eps):
    """ValueError for what orthogonalize refuses: the library looks at it before it looks at matrices, of which there are none."""
    key = (int(steps), repr(coefficients), float(eps))
    if key in _TAKEN:
        return
    if not 1 <= key[0] <= 16:
        raise ValueError(f"steps must be in [1, 16] (got {steps})")
    table = _table(key[0], coefficients)
    if type(table) is not torch.Tensor:             # under FakeTensorMode: without values there is nothing to look at
        return
    L = _native.lib()
    if L.mace_b200_orthogonalize(None, 1, 1, None, None, 0, 1, 1, table.data_ptr(), key[0], key[2], 0, None):
        raise ValueError(L.mace_b200_last_error().decode())
    if len(_TAKEN) > 64:
        _TAKEN.clear()
    _TAKEN.add(key)


def orthogonalize(g, *, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """g [.., m, n] (float32, bfloat16 or float16) -> bfloat16 [.., m, n]: X = g / (|g| + eps) with the Frobenius norm, then `steps`
    times X = a X + (b A + c A A) X with A = X X^T (from the right with A = X^T X for m > n).  Every matrix of the batch for itself.

    coefficients: (a, b, c), or a triple for each step; what they do to singular values in (0, 1] must stay below 3.5.
    Products take operands rounded to float16 (X itself and the diagonals stay in float32): the result is off by 2e-4 to 1.2e-3 of its
    norm before it is rounded to bfloat16, which adds 1.7e-3, whatever the type of g (2 x 2 matrices by 2e-3, rarely by 1%).
    The last two dimensions' rows may be strided.  At most 16 steps and sides of 65,536.  No gradient."""
    steps = int(steps)
    if not 1 <= steps <= 16:
        raise ValueError(f"steps must be in [1, 16] (got {steps})")
    return _op("orthogonalize")(g, _table(steps, coefficients), float(eps))


class Muon(torch.optim.Optimizer):
    """Momentum whose update of a matrix [.., m, n] is orthogonalised: p <- p (1 - lr weight_decay) - lr max(1, m / n)^0.5 U with
    U = orthogonalize(g + momentum v) (nesterov) or of v, and v <- momentum v + g.  For parameters of two dimensions or more;
    vectors (norms, biases) take another optimiser.

    All of it is float32 whatever the parameter's type.  A bfloat16 or float16 parameter keeps what its rounding left off beside v
    ("rounding"), p + rounding being the float32 value that the step goes on from: updates and decays below half a step of the type
    add up, and a parameter that is set from outside stays set."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group):
        """ValueError for a group that a step would refuse."""
        lr, momentum, weight_decay = group["lr"], group["momentum"], group["weight_decay"]
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError(f"lr {lr}, momentum {momentum} or weight_decay {weight_decay} is out of range")
        _check_polynomial(group["steps"], group["coefficients"], group["eps"])
        for p in group["params"]:
            if p.dim() < 2:
                raise ValueError(f"Muon takes matrices [.., m, n] (got a parameter of shape {tuple(p.shape)})")
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise ValueError(f"Muon takes float32, bfloat16 or float16 parameters (got {p.dtype})")
            if max(p.shape[-2:]) > 65536 or p.shape[:-2].numel() > 65535:
                raise ValueError(f"Muon takes at most 65535 matrices with sides of at most 65536 (got {tuple(p.shape)})")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:              # before any state changes: groups may be edited between steps
            self._check(group)
            for p in group["params"]:
                if p.grad is not None and (not p.is_cuda or p.grad.is_sparse):
                    raise ValueError("Muon takes CUDA parameters with dense gradients")
        for group in self.param_groups:
            lr, mu = group["lr"], group["momentum"]
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                state, narrow = self.state[p], p.dtype != torch.float32
                for key in ("momentum_buffer", "rounding")[:1 + narrow]:
                    if key not in state:
                        state[key] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                v = state["momentum_buffer"]
                v.mul_(mu).add_(p.grad)
                d = p.grad.float().add(v, alpha=mu) if group["nesterov"] else v
                u = orthogonalize(d, steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
                w = p.float().add_(state["rounding"]) if narrow else p
                if group["weight_decay"]:
                    w.mul_(1 - lr * group["weight_decay"])
                w.add_(u, alpha=-lr * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5)
                if narrow:
                    p.copy_(w)
                    torch.sub(w, p, out=state["rounding"])
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class has cast the state to the parameters' types
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(ids, [p for group in self.param_groups for p in group["params"]]):
            for key, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value) and value.is_floating_point():
                    self.state[p][key] = value.to(device=p.device, dtype=torch.float32, copy=True)
