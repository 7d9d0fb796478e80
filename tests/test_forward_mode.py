"""Forward-mode derivatives of layer norm, routing and expert products are refused (shape tensors: no kernel runs)."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

from mace_onegpu import _native as N

CALLS = {
    "layer_norm x": (lambda o, d: o.layer_norm(d(6, 16), None, None, 1e-5)),
    "layer_norm weight": (lambda o, d: o.layer_norm(torch.empty(6, 16, device="cuda"), d(16), None, 1e-5)),
    "layer_norm bias": (lambda o, d: o.layer_norm(torch.empty(6, 16, device="cuda"), None, d(16), 1e-5)),
    "route logits": (lambda o, d: o.route(d(6, 8), None, 2, True, 1, 1, True, 1.0)),
    "expert_linear x": (lambda o, d: o.expert_linear(d(6, 16), torch.empty(4, 5, 16, device="cuda"), _ex(), None, None)),
    "expert_linear w": (lambda o, d: o.expert_linear(torch.empty(6, 16, device="cuda"), d(4, 5, 16), _ex(), None, None)),
    "expert_linear weights": (lambda o, d: o.expert_linear(torch.empty(6, 16, device="cuda"), torch.empty(4, 5, 16, device="cuda"),
                                                           _ex(), None, d(6, 2))),
}


def _ex():
    return torch.empty(6, 2, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("grad", [False, True])
def test_dual_tensors_are_refused(name, grad):
    ops = N.ops()
    with FakeTensorMode(), fw.dual_level():
        def dual(*shape):
            return fw.make_dual(torch.empty(*shape, device="cuda", requires_grad=grad), torch.empty(*shape, device="cuda"))

        assert fw.unpack_dual(dual(3) * 2).tangent is not None
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[name](ops, dual)


def test_jvp_is_refused():
    ops = N.ops()
    with FakeTensorMode():
        x = torch.empty(6, 16, device="cuda")
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(lambda t: ops.layer_norm(t, None, None, 1e-5), (x,), (x,))


def test_plain_tensors_inside_a_dual_level_pass():
    ops = N.ops()
    with FakeTensorMode(), fw.dual_level():
        assert ops.layer_norm(torch.empty(6, 16, device="cuda"), None, None, 1e-5).shape == (6, 16)
        # the bias of route only ranks: its derivative is zero, and nothing is lost
        b = fw.make_dual(torch.empty(8, device="cuda"), torch.empty(8, device="cuda"))
        assert ops.route(torch.empty(6, 8, device="cuda"), b, 2, True, 1, 1, True, 1.0)[0].shape == (6, 2)
