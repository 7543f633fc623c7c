"""Device batch sizes with an empty contraction (dim 0): the used rows are 0, the others left as they were."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


def call(sizes, cap, dim_out, dtype, swiglu, int8, d):
    from gmm_b200 import capi
    lib = capi.load()
    bs = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    one = torch.ones(max(cap, len(sizes) * dim_out), device="cuda")
    if int8:
        rc = lib.gmm_sm100_forward_int8_dev(None, one.data_ptr(), None, one.data_ptr(), bs.data_ptr(), len(sizes), cap, 0,
                                            dim_out, capi.dtype_code(dtype), swiglu, d.data_ptr(), None)
    else:
        rc = lib.gmm_sm100_forward_dev(None, None, bs.data_ptr(), len(sizes), cap, 0, dim_out, capi.dtype_code(dtype), 0,
                                       swiglu, d.data_ptr(), None, 0, None)
    torch.cuda.synchronize()
    return rc


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype,swiglu", [(torch.bfloat16, 0), (torch.float16, 1), (torch.float32, 0)])
@pytest.mark.parametrize("sizes,cap", [([2, 0, 3], 9), ([0, 0], 4), ([1], 1), ([700, 0, 1, 512], 1300), ([1] * 1024, 1024)])
def test_rows_behind_the_last_are_left(sizes, cap, dtype, swiglu, int8):
    dim_out = 48
    d = torch.full((cap, dim_out // 2 if swiglu else dim_out), 7.0, dtype=dtype, device="cuda")
    assert call(sizes, cap, dim_out, dtype, swiglu, int8, d) == 0
    used = sum(sizes)
    assert (d[:used] == 0).all() and (d[used:] == 7).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("sizes,status", [([4, 3], -2), ([-1, 3], -1), ([2 ** 31 - 1, 2 ** 31 - 1], -2)])
def test_bad_sizes_are_recorded(sizes, status, int8):
    from gmm_b200 import capi
    d = torch.full((6, 16), 7.0, device="cuda")
    assert call(sizes, 6, 16, torch.float32, 0, int8, d) == 0
    assert capi.device_error(clear=True) == status
    assert (d == 7).all()
