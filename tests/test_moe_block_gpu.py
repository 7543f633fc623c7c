"""An MoE block of a model whose parameters require gradients: served without a graph, refused with one."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


@pytest.mark.parametrize("int8", [False, True])
def test_parameters_that_require_gradients(int8):
    from gmm_b200.int8 import quantize_experts
    from gmm_b200.moe import moe_block
    from gmm_b200.norms import pre_norm
    g = torch.Generator().manual_seed(1)
    T, dim, inter, E = 9, 64, 32, 4
    x = torch.randn(T, dim, generator=g).bfloat16().cuda()
    w1, w2 = ((torch.randn(*s, generator=g) / 8).bfloat16().cuda() for s in ((E, dim, 2 * inter), (E, inter, dim)))
    if int8:
        w1, w2 = quantize_experts(w1), quantize_experts(w2)
    router, norm = (torch.randn(*s, generator=g).bfloat16().cuda() for s in ((dim, E), (dim,)))
    want = moe_block(x, pre_norm(x, norm), router, w1, w2, 2, norm, next_weight=norm)
    for p in (router, norm):
        p.requires_grad_()
    with torch.no_grad():
        got = moe_block(x, pre_norm(x, norm), router, w1, w2, 2, norm, next_weight=norm)
    with torch.inference_mode():
        again = moe_block(x, pre_norm(x, norm), router, w1, w2, 2, norm, next_weight=norm)
    for a, b, c in zip(got, again, want):
        assert not a.requires_grad and torch.equal(a, c) and torch.equal(b, c)
    with pytest.raises(RuntimeError, match="no backward pass"):
        moe_block(x, pre_norm(x, norm), router, w1, w2, 2, norm)
