"""Row quantiser at the widths where its shared memory is fullest."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    from gmm_b200 import capi
    assert capi.device_error(clear=True) == 0


def exact(x):
    """Codes and scales as defined: two fp32 divisions, correctly rounded, which torch's CPU divisions are."""
    x = x.float()
    scale = x.abs().amax(1) / torch.full((x.shape[0],), 127.0)
    return torch.round(x / scale[:, None]).to(torch.int8), scale


# every band of widths in which the number of row slots changes, in whole words and off them
@pytest.mark.parametrize("dim", [8192, 8200, 10920, 10928, 12616, 12624, 12625, 12630, 12632, 12640, 12648, 12652, 12656, 12664,
                                 14000, 16229, 16232, 16240, 16241, 16248, 16256, 16264, 16272, 16280, 16383, 16384, 16385])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_rows(dim, dtype):
    from gmm_b200.int8 import quantize_rows
    x = (torch.randn(7, dim, generator=torch.Generator().manual_seed(dim)) * 3).to(dtype)
    q, s = quantize_rows(x.cuda())
    codes, scale = exact(x)
    assert torch.equal(s.cpu(), scale)
    assert torch.equal(q[:, :dim].cpu(), codes) and (q[:, dim:] == 0).all()


def test_expert_weights_of_a_wide_contraction():
    from gmm_b200.int8 import quantize_experts
    w = torch.randn(2, 12640, 8, generator=torch.Generator().manual_seed(1))
    q, s = quantize_experts(w.cuda())
    codes, scale = exact(w.transpose(1, 2).reshape(16, 12640))
    assert torch.equal(s.cpu().flatten(), scale) and torch.equal(q.cpu().view(16, -1), codes)
