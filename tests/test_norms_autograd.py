"""What the norms and the block around them differentiate, without a GPU: on fake CUDA tensors the operators' autograd
runs as it does on real ones, with no kernel below it."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

NAMES = ("y", "x", "w", "g", "v")


def norm_inputs():
    shapes = {"y": (6, 40), "x": (6, 40), "w": (40,), "g": (6, 1), "v": (40,)}
    return {k: torch.empty(s, device="cuda") for k, s in shapes.items()}


def run(t):
    from gmm_b200.norms import post_norm
    return post_norm(t["y"], t["x"], t["w"], gate=t["g"], gate_act="tanh", next_weight=t["v"])


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", NAMES)
def test_a_forward_gradient_is_refused(which, grad_mode, requires_grad):
    with FakeTensorMode(), torch.set_grad_enabled(grad_mode), fwAD.dual_level():
        t = norm_inputs()
        t[which] = fwAD.make_dual(t[which].requires_grad_(requires_grad), torch.empty_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            run(t)


def test_functional_forward_transforms_are_refused():
    from gmm_b200.norms import pre_norm
    with FakeTensorMode():
        t = norm_inputs()
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(lambda a: pre_norm(a, t["w"]), (t["x"],), (t["y"],))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jacfwd(lambda a: pre_norm(t["x"], a))(t["w"])


def test_the_backward_operator_refuses_a_forward_gradient():
    """Forward over reverse: the gradient that comes in is a dual tensor."""
    with FakeTensorMode(), torch.no_grad(), fwAD.dual_level():
        t = norm_inputs()
        stats = torch.empty(2, 6, device="cuda")
        dx = fwAD.make_dual(torch.empty(6, 40, device="cuda"), torch.empty(6, 40, device="cuda"))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.ops.hopper_gmm_fwd.post_norm_backward(t["y"], t["x"], t["w"], t["g"], t["v"], stats, dx, None, 1, 1.0, 0.0)


def test_plain_tensors_inside_a_dual_level_run():
    with FakeTensorMode(), fwAD.dual_level():
        t = norm_inputs()
        assert run(t)[0].shape == (6, 40)
        t["x"].requires_grad_()
        assert run(t)[1].requires_grad


# ------------------------------------------------------------------ the block between the norms
BLOCK = ("x", "h", "router", "gate_up", "down", "post", "next", "gate")


def block_inputs(int8):
    shapes = {"x": (6, 48), "h": (6, 48), "router": (48, 4), "post": (48,), "next": (48,), "gate": (48,)}
    t = {k: torch.empty(s, dtype=torch.bfloat16, device="cuda") for k, s in shapes.items()}
    if int8:
        t["gate_up"] = (torch.empty(4, 64, 48, dtype=torch.int8, device="cuda"), torch.empty(4, 64, device="cuda"))
        t["down"] = (torch.empty(4, 48, 32, dtype=torch.int8, device="cuda"), torch.empty(4, 48, device="cuda"))
    else:
        t["gate_up"] = torch.empty(4, 48, 64, dtype=torch.bfloat16, device="cuda")
        t["down"] = torch.empty(4, 32, 48, dtype=torch.bfloat16, device="cuda")
    return t


def block(t):
    from gmm_b200.moe import moe_block
    return moe_block(t["x"], t["h"], t["router"], t["gate_up"], t["down"], 2, t["post"], next_weight=t["next"], gate=t["gate"])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("which", BLOCK)
def test_a_block_refuses_gradients_it_would_drop(which, int8):
    """Its expert layer keeps no graph, while the norm after it would: a gradient from it would lack the experts' part."""
    with FakeTensorMode():
        t = block_inputs(int8)
        (t[which][1] if isinstance(t[which], tuple) else t[which]).requires_grad_()
        t["down"] = list(t["down"]) if int8 else t["down"]  # a pair is any sequence of two
        with pytest.raises(RuntimeError, match="no backward pass"):
            block(t)


@pytest.mark.parametrize("which", BLOCK)
def test_a_block_refuses_forward_gradients(which):
    with FakeTensorMode(), torch.no_grad(), fwAD.dual_level():
        t = block_inputs(False)
        t[which] = fwAD.make_dual(t[which], torch.empty_like(t[which]))
        with pytest.raises(RuntimeError, match="no backward pass"):
            block(t)


def test_quantised_parameters_carry_no_graph():
    """The codes and scales of parameters go into a block like any others."""
    from gmm_b200.int8 import quantize_experts
    with FakeTensorMode():
        w = torch.empty(4, 48, 64, device="cuda", requires_grad=True)
        for t in quantize_experts(w) + quantize_experts(w, trans_b=True):
            assert not t.requires_grad and t.grad_fn is None
