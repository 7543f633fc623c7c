"""The norms under torch.compile: traced through the fake implementations, forward and backward."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("use_h", [True, False])
def test_compiled_step(backend, use_h):
    """The same kernels on the same inputs: equal results, whatever of h is used."""
    from gmm_b200.norms import post_norm, pre_norm
    g = torch.Generator().manual_seed(1)
    shapes = ((6, 40), (6, 40), (40,), (6, 1), (40,))
    t = [torch.randn(*s, generator=g).cuda().requires_grad_() for s in shapes]

    def step(y, x, w, gate, v):
        new, h = post_norm(y, x, w, gate=gate, gate_act="tanh", residual_scale=0.5, next_weight=v)
        return (new * new).sum() + ((h * h).sum() if use_h else 0) + pre_norm(x, v).sum()

    want = torch.autograd.grad(step(*t), t)
    torch._dynamo.reset()
    got = torch.autograd.grad(torch.compile(step, backend=backend, fullgraph=True)(*t), t)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_operator_registration():
    from torch.library import opcheck
    import gmm_b200  # noqa: F401
    y, x = (torch.randn(6, 40, device="cuda", requires_grad=True) for _ in range(2))
    w, v = (torch.randn(40, device="cuda", requires_grad=True) for _ in range(2))
    opcheck(torch.ops.hopper_gmm_fwd.post_norm.default, (y, x, w, None, v, 0, 0.5, 1e-6, 0.0, False))
