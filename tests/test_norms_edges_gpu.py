"""Norms where a gradient is finite beside an infinity."""

import pytest
import torch

from test_norms_gpu import check, cuda, formulas, inputs, train

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    from gmm_b200 import capi
    assert capi.device_error(clear=True) == 0


# ------------------------------------------------------------------ no gradient of h
@pytest.mark.parametrize("following", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(5, 24), (400, 33), (9, 4096), (4, 8200), (3, 9001)])
def test_without_a_gradient_of_h_the_residual_has_no_part(T, D, dtype, gate, following):
    """dx is dx' itself, and dy, dw and dg do not depend on x: an infinity or NaN in it stays out of them."""
    d = inputs(T, D, dtype, torch.float32, gate, following, seed=31)
    want = formulas(d, "tanh", 0.7, use_dh=False)
    d["x"][0] = float("inf")
    d["x"][1, D // 2] = float("nan")
    d["x"][2, D - 1] = float("-inf")
    got = train(cuda(d), "tanh", 0.7, use_dh=False)
    assert torch.equal(got["dx"].cpu(), d["dx"])
    for k in ("dy", "dw") + (() if gate == "none" else ("dg",)):
        check(got[k], want[k], k)
    if following:
        assert (got["dv"] == 0).all()


def test_without_a_gradient_of_h_a_spoilt_y_leaves_dx():
    d = inputs(4, 40, torch.float32, gate="full", following=False, seed=32)
    d["y"][1, 3], d["y"][2, 5], d["g"][3, 7] = float("nan"), float("inf"), float("inf")
    got = train(cuda(d), "none", 0.7)
    assert torch.equal(got["dx"].cpu(), d["dx"])
    assert got["dy"][1].isnan().all() and not got["dy"][0].isnan().any()
