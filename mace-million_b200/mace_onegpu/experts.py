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


def _stream(index):
    """Handle of the current stream of CUDA device `index` (a Stream object would cost a small call 2 us); 0 elsewhere."""
    return torch._C._cuda_getCurrentRawStream(index) if index >= 0 and torch.cuda.is_initialized() else 0


def _place(index):
    """The current stream and the number of the CUDA graph capture it is in (0: none)."""
    stream = _stream(index)
    return stream, N.lib().mace_b200_capture_id(stream) if index >= 0 and torch.cuda.is_initialized() else 0


def _ready(device):
    """An event of what the current stream holds so far."""
    return torch.cuda.current_stream(device).record_event()


def _after(device, event, *tensors):
    """Makes the current stream wait for the event, and the tensors live for as long as it uses them."""
    stream = torch.cuda.current_stream(device)
    if event is not None:
        stream.wait_event(event)
    for t in tensors:
        t.record_stream(stream)


class ExpertPlan:
    """The slots (token, choice) of `experts` [T, k] (or [T]) in expert order, for any number of expert_linear calls
    with the same choice.  An expert of -1 means none.

    Contiguous int32 indices are kept as they are (a copy would cost a small call half of its time): products refuse a plan
    whose indices torch has changed since.  Others are copied.  They are sorted at the first product that needs it, and
    products on other streams wait for that.  A CUDA graph sorts for itself, at every replay what the indices' buffer holds
    then; nothing sorted in a capture is used outside of it.  Where a graph's replays write the indices, make a new plan
    after each (nothing tells an older one), or make it in the graph."""

    def __init__(self, experts, n_experts):
        n = experts.dim()
        if n not in (1, 2) or experts.dtype not in (torch.int32, torch.int64):
            raise ValueError("experts must be an integer tensor [tokens, k] or [tokens]")
        self.n_experts = int(n_experts)
        if self.n_experts < 1:
            raise ValueError("n_experts must be positive")
        if n == 1:
            experts = experts[:, None]
        mine = True                                 # a copy of the caller's indices
        if experts.dtype != torch.int32:
            # 64-bit indices outside the range of int32 must not wrap into it: -2 is refused by check(), like any other
            experts = torch.where((experts >= -1) & (experts < self.n_experts), experts, -2).to(torch.int32).contiguous()
        elif not experts.is_contiguous():
            experts = experts.contiguous()
        elif experts.is_inference():                # has no version
            experts = experts.clone()
        else:
            mine = False
        self.experts = experts
        self._start(None if mine else experts._version)

    def _start(self, version):
        self._version = version
        self._index = self.experts.get_device()
        self._stream, self._capture = _place(self._index)
        self._sorted = None                         # (words, stream, capture, event)

    def __getstate__(self):                         # copies and saved plans sort for themselves
        return {"experts": self.experts, "n_experts": self.n_experts}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._start(None if self.experts.is_inference() else self.experts._version)

    def use(self, stream):
        """Checks that the indices are the ones that the plan was made of, and keeps them alive for that stream."""
        if self._version is not None and self.experts._version != self._version:
            raise RuntimeError("the indices of this plan were changed in place after plan_experts: make a new plan")
        if stream != self._stream:
            _after(self.experts.device, None, self.experts)

    @property
    def words(self):
        """The plan as the kernels read it (int32), for the current stream."""
        stream, capture = _place(self._index)
        self.use(stream)
        s = self._sorted
        # tables of another capture hold nothing before its first replay; eager ones may be freed while a graph uses them;
        # and the indices of a plan that was made in a capture are written anew by every replay
        if s is None or s[2] != capture or (capture == 0 and self._capture != 0):
            s = (_op("expert_plan")(self.experts, self.n_experts), stream, capture, _ready(self.experts.device))
            self._sorted = s
        elif s[1] != stream:
            _after(self.experts.device, s[3], s[0])
        return s[0]

    def check(self):
        """Reads the device status word (synchronises) and raises if an index was outside [-1, n_experts) or a product
        outside of CUDA graphs gave up waiting."""
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
    None: out [T, k, O] = w[e_tj] x.  x and w: float32 (at fp32 accuracy; infinities come out as NaN), bfloat16 or float16
    (results rounded once).  Slots with expert -1 give zeros and no gradient.  Differentiable w.r.t. x, w and weights; sums
    run in a fixed order."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError("plan must be an ExpertPlan (plan_experts(experts, n_experts))")
    if w.dim() != 3 or w.shape[0] != plan.n_experts:
        raise ValueError(f"w must be [{plan.n_experts}, out, in] (got {tuple(w.shape)})")
    slots = plan.experts.numel()
    few = slots <= FEW_SLOTS and slots * w.shape[1] * w.shape[2] * w.element_size() <= FEW_BYTES
    if few and torch.is_grad_enabled():
        few = not (x.requires_grad or w.requires_grad or (weights is not None and weights.requires_grad))
    if few:
        plan.use(_stream(plan._index))
    return _op("expert_linear")(x, w, plan.experts, None if few else plan.words, weights)


class ExpertBlock(torch.nn.Module):
    """Layer norm, router and a two-layer expert network per atom: out_t = sum_j g_tj W2[e_tj] silu(W1[e_tj] norm(x_t)).

    x [T, dim] (rows may be strided) -> [T, out].  The router's bias (a buffer) only ranks; `balance` moves it towards
    an even load after a step, so no loss term is needed for it."""

    def __init__(self, dim, hidden, out, n_experts, k, score="sigmoid", dtype=torch.float32, device="cuda", seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)

        def par(*shape, scale):
            return torch.nn.Parameter((torch.randn(*shape, generator=g) * scale).to(device=device, dtype=dtype))

        self.n_experts, self.k, self.score = int(n_experts), int(k), score
        self.gamma = torch.nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.beta = torch.nn.Parameter(torch.zeros(dim, device=device, dtype=dtype))
        self.router = par(n_experts, dim, scale=dim ** -0.5)
        self.w1 = par(n_experts, hidden, dim, scale=dim ** -0.5)
        self.w2 = par(n_experts, out, hidden, scale=hidden ** -0.5)
        self.register_buffer("bias", torch.zeros(n_experts, device=device))
        self.plan = None                            # of the last forward call

    def forward(self, x):
        xn = layer_norm(x, self.gamma, self.beta)
        weights, experts = route(xn @ self.router.T, self.k, bias=self.bias, score=self.score)
        self.plan = plan = plan_experts(experts, self.n_experts)
        h = torch.nn.functional.silu(expert_linear(xn, self.w1, plan))
        return expert_linear(h, self.w2, plan, weights)

    @torch.no_grad()
    def balance(self, rate=1e-3):
        """Raises the bias of experts that got less than the mean load in the last call, lowers the others'."""
        load = torch.bincount(self.plan.experts.flatten() + 1, minlength=self.n_experts + 1)[1:].float()
        self.bias += rate * torch.sign(load.mean() - load)
        return load


def water_features(n, dtype, seed=0):
    """Layer-1 scalar features H1[:, 0e] [3 n^3, 128] (rows 512 apart) of a water box under the random-init model, and the model's
    per-atom energies [3 n^3, 1], centred and scaled to deviation one."""
    from . import model as M
    from . import neighbors, structures
    from .engine import ThreePassEngine

    mdl = M.default_model(seed)
    pos, Z, box = structures.water_box(n, seed=seed)
    cols = structures.species_columns(Z, mdl.arch.atomic_numbers)
    pi, pj, rij = neighbors.neighbor_list(pos, box, mdl.arch.r_max)
    eng = ThreePassEngine(mdl, sorted(set(cols.tolist())), chunk=min(16384, len(Z)), device="cuda")
    plan = eng.plan(pi, pj, rij, torch.as_tensor(cols), len(Z), len(Z))
    eat, _ = eng.evaluate(plan)
    h1 = eng.node_features(plan)
    e = eat.double()
    target = ((e - e.mean()) / e.std()).float()[:, None].to(dtype)
    return h1.to(dtype)[:, 0], target


class _Together:
    """Several optimisers as one."""

    def __init__(self, *opts):
        self.opts = opts

    def zero_grad(self):
        for o in self.opts:
            o.zero_grad()

    def step(self):
        for o in self.opts:
            o.step()


def train_readout(n=8, n_experts=8, k=2, hidden=64, steps=200, lr=3e-3, dtype=torch.float32, seed=0, optimizer="adam",
                  lr_matrices=0.02):
    """Trains an ExpertBlock to give the per-atom energies of the model from its layer-1 scalar features H1[:, 0e] of a
    water box of 3 n^3 atoms (random-init weights).  optimizer: "adam", or "muon" for the experts' matrices and the router (with
    lr_matrices) and Adam for the rest.  Returns a dict of what happened."""
    import time

    if optimizer not in ("adam", "muon"):
        raise ValueError(f"optimizer must be 'adam' or 'muon' (got {optimizer!r})")
    x, target = water_features(n, dtype, seed)
    block = ExpertBlock(128, hidden, 1, n_experts, k, dtype=dtype, seed=seed)
    if optimizer == "muon":
        from . import optim

        opt = _Together(optim.Muon([p for p in block.parameters() if p.dim() >= 2], lr=lr_matrices),
                        torch.optim.Adam([p for p in block.parameters() if p.dim() < 2], lr=lr))
    else:
        opt = torch.optim.Adam(block.parameters(), lr=lr)
    losses = []
    t0 = time.perf_counter()
    for _ in range(steps):
        opt.zero_grad()
        loss = torch.nn.functional.mse_loss(block(x).float(), target.float())
        loss.backward()
        opt.step()
        load = block.balance(1e-2)
        losses.append(loss.detach())
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    block.plan.check()
    return {"atoms": len(x), "experts": n_experts, "k": k, "steps": steps, "dtype": str(dtype).split(".")[-1],
            "loss_first": float(losses[0]), "loss_last": float(losses[-1]), "steps_per_s": steps / dt,
            "load": [int(v) for v in load.tolist()]}


def main():
    import argparse
    import json

    ap = argparse.ArgumentParser(description="Train a mixture-of-experts readout over layer-1 features of a water box")
    ap.add_argument("--n", type=int, default=8, help="molecules along an edge (3 n^3 atoms)")
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--k", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=64)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--dtype", default="float32", choices=["float32", "bfloat16", "float16"])
    ap.add_argument("--optimizer", default="adam", choices=["adam", "muon"], help="muon: for the matrices, Adam for the rest")
    ap.add_argument("--lr-matrices", type=float, default=0.02, help="of the matrices with --optimizer muon")
    a = ap.parse_args()
    print(json.dumps(train_readout(a.n, a.experts, a.k, a.hidden, a.steps, a.lr, getattr(torch, a.dtype), optimizer=a.optimizer,
                                   lr_matrices=a.lr_matrices)))


if __name__ == "__main__":
    main()
