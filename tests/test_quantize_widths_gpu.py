"""Row quantiser at the widths where its shared memory is fullest, and at the ends of its buffers."""

import pytest
import torch

from test_norms_edges_gpu import Guarded, code

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,dim", [(1, 1), (700, 17), (301, 250), (5, 4096), (3, 16381), (2, 20000)])
def test_nothing_is_written_outside(T, dim, dtype):
    from gmm_b200 import capi
    lib = capi.load()
    x = torch.randn(T, dim, generator=torch.Generator().manual_seed(2)).to(dtype)
    c = x.cuda()
    k = 2
    place = torch.randperm(T * k, generator=torch.Generator().manual_seed(3)).view(T, k).int()
    out = Guarded()
    q, q_t = out.empty((T * k, (dim + 15) // 16 * 16), torch.int8)
    s, s_t = out.empty((T * k,), torch.float32)
    dst = place.cuda()
    rc = lib.gmm_sm100_quantize_rows(c.data_ptr(), code(dtype), T, dim, dst.data_ptr(), k, T * k, q, s, None)
    assert rc == 0, lib.gmm_sm100_last_error()
    out.check()
    codes, scale = exact(x)
    want = torch.zeros(T * k, (dim + 15) // 16 * 16, dtype=torch.int8)
    want_s = torch.empty(T * k)
    for j in range(k):
        want[place[:, j].long(), :dim] = codes
        want_s[place[:, j].long()] = scale
    assert torch.equal(q_t().cpu(), want) and torch.equal(s_t().cpu(), want_s)
