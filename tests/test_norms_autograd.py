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
