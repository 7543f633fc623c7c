"""Norms where a gradient is finite beside an infinity and where a gate saturates, and at the ends of their buffers."""

import pytest
import torch

from test_norms_gpu import HALF_STEP, H, TINY, check, cuda, formulas, inputs, train

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


# ------------------------------------------------------------------ gates
# Rows of y = 1 with eps = 0 and a power of two elements have mean 1 exactly, so r(y) is 1 within rsqrtf's 2 ulp (4 h).
GATES = [0.0, 0.3, 0.5, 1.0, 2.0, 3.3, 4.0, 6.7, 8.0, 10.0, 12.0, 14.1, 16.0, 20.0, 30.0]


def gate_values(dtype, n):
    g = torch.tensor([s * v for v in GATES for s in (1, -1)] + [float("inf"), float("-inf")])
    spread = (torch.rand(n - g.numel(), generator=torch.Generator().manual_seed(41)) * 2 - 1) * 30
    return torch.cat([g, spread]).to(dtype)


def gate_exact(g, kind):
    """act(g) and act'(g) in fp64, neither from the other by a difference."""
    g = g.double()
    if kind == "sigmoid":
        e = torch.exp(-g.abs())
        return torch.where(g >= 0, 1 / (1 + e), e / (1 + e)), e / (1 + e) ** 2
    e = torch.exp(-2 * g.abs())
    return torch.tanh(g), 4 * e / (1 + e) ** 2


def gate_case(gate, dtype, gate_dtype, kind):
    """x_new and dgate of rows of ones (x = 0, w = 1, dx' = 1): act(g), and D or T times act'(g) where g is shared."""
    from gmm_b200.norms import post_norm
    T, D = {"channel": (1, 1024), "token": (1024, 8), "full": (8, 1024)}[gate]
    g = gate_values(gate_dtype, 1024)
    shape = {"channel": (D,), "token": (T, 1), "full": (T, D)}[gate]
    g = g.repeat(8).view(T, D) if gate == "full" else g.view(shape)
    y = torch.ones(T, D, dtype=dtype, device="cuda", requires_grad=True)
    x, w = torch.zeros(T, D, dtype=dtype, device="cuda"), torch.ones(D, device="cuda")
    leaf = g.cuda().requires_grad_()
    new = post_norm(y, x, w, gate=leaf, gate_act=kind, eps=0.0)
    dg, = torch.autograd.grad(new, leaf, torch.ones_like(new))
    a, da = gate_exact(g, kind)
    return new, a.expand(T, D), dg, da * (D if gate == "token" else 1)


def near(got, want, rel, what):
    tol = want.abs() * (rel + HALF_STEP[got.dtype] * (1 + 2.0 ** -8)) + TINY[got.dtype]
    off = (got.detach().double().cpu() - want).abs()
    worst = (off / tol).argmax()
    assert (off <= tol).all(), (what, float((off / tol).max()), int(worst))


GATES_OF = pytest.mark.parametrize("gate", ["channel", "token", "full"])
KINDS = pytest.mark.parametrize("kind", ["tanh", "sigmoid"])


@GATES_OF
@KINDS
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_act_of_fp32_gates(dtype, kind, gate):
    """An fp32 gate beside rows of any type: act(g) within 14 h of its value at any |g|.  The exponential 2 ulp (4 h), the
    sum, the quotient and a product h each, or tanhf 2 ulp; r(y) 4 h and three products."""
    new, a, _, _ = gate_case(gate, dtype, torch.float32, kind)
    near(new, a, 14 * H, "act")


@GATES_OF
@KINDS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_act_of_16_bit_gates(dtype, kind, gate):
    """The fast exponential of x is within 2 + 1.173 |x| ulp, 75 h at |x| = 30, the fast quotient 2 ulp, the rest as above."""
    new, a, _, _ = gate_case(gate, dtype, dtype, kind)
    near(new, a, 100 * H, "act")


@GATES_OF
@KINDS
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_slope_of_fp32_gates(dtype, kind, gate):
    """act'(g) within 24 h of its value, however far the gate is saturated: the exponential 4 h, 1 + e and its square 3 h,
    the quotients and products 3 h; r(y) 4 h, the products with pw, y and dx' 4 h, and the sum over equal elements of a
    row 3 h (channel: one row)."""
    _, _, dg, da = gate_case(gate, dtype, torch.float32, kind)
    near(dg, da, 24 * H, "slope")


@GATES_OF
@KINDS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_slope_of_16_bit_gates(dtype, kind, gate):
    """The fast exponential of x is within 146 h for |x| = 60 (tanh's slope at |g| = 30), and the rest of the slope less than
    40 h; the gradient's own half step (2^-11 and more) is above both."""
    _, _, dg, da = gate_case(gate, dtype, dtype, kind)
    near(dg, da, 200 * H, "slope")


@GATES_OF
@KINDS
def test_no_slope_at_infinite_gates(gate, kind):
    _, _, dg, _ = gate_case(gate, torch.float32, torch.float32, kind)
    at = gate_values(torch.float32, 1024).isinf()
    dg = dg.flatten()[:1024].cpu()
    assert (dg[at] == 0).all() and not dg.isnan().any()


@pytest.mark.parametrize("D", [1, 24])
def test_a_token_gate_of_one_row_without_batch_dimensions(D):
    """[..., 1] with no leading dimension is [1]."""
    from gmm_b200.norms import post_norm
    d = inputs(1, D, torch.float32, gate="token", following=False, seed=33)
    want = formulas(d, "sigmoid", 0.6)
    c = cuda(d)
    leaves = {k: (c[k][0] if k != "w" else c[k]).detach().clone().requires_grad_() for k in ("y", "x", "w", "g")}
    new = post_norm(leaves["y"], leaves["x"], leaves["w"], gate=leaves["g"], gate_act="sigmoid", residual_scale=0.6)
    grads = torch.autograd.grad(new, list(leaves.values()), c["dx"][0])
    check(new, (want["new"][0][0], want["new"][1][0]), "new")
    for k, gr in zip(leaves, grads):
        value, bound = want["d" + k]
        check(gr, (value.reshape(gr.shape), bound.reshape(gr.shape)), k)


# ------------------------------------------------------------------ the ends of the buffers
GUARD = 512
FILL = 0xA5


class Guarded:
    """Buffers between guard regions; an output starts `shift` bytes off a 16-byte word and ends with its last byte."""

    def __init__(self):
        self.made = []

    def empty(self, shape, dtype, shift=0):
        size = torch.empty(0, dtype=dtype).element_size()
        n = size
        for s in shape:
            n *= s
        raw = torch.full((GUARD + shift + n + GUARD,), FILL, dtype=torch.uint8, device="cuda")
        self.made.append((raw, GUARD + shift, n))
        view = raw[GUARD + shift: GUARD + shift + n]
        return raw.data_ptr() + GUARD + shift, lambda: view.clone().view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for i, (raw, at, n) in enumerate(self.made):
            assert (raw[:at] == FILL).all(), ("before buffer", i)
            assert (raw[at + n:] == FILL).all(), ("behind buffer", i)


def code(t):
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[t]


@pytest.mark.parametrize("off", [False, True])
@pytest.mark.parametrize("gate,gate_dtype", [("none", None), ("channel", torch.float32), ("channel", None),
                                             ("token", None), ("full", None), ("full", torch.float32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", [(1, 1), (300, 3), (700, 11), (5, 33), (400, 250), (160, 2050), (9, 4091), (3, 4096),
                                 (151, 8195), (2, 16363), (3, 16384)])
def test_nothing_is_written_outside(T, D, dtype, gate, gate_dtype, off):
    """Forward and backward through the C entry points, every output and the workspace between guards; the results
    are those of tensors of their own."""
    from gmm_b200 import capi
    lib = capi.load()
    gate_dtype = gate_dtype or dtype
    d = inputs(T, D, dtype, torch.float32, gate, seed=51)
    if d["g"] is not None:
        d["g"] = d["g"].to(gate_dtype)
    c = cuda(d)
    want = train(c, "tanh", 0.7)
    mode = ["none", "channel", "token", "full"].index(gate if gate != "token" or D > 1 else "full")  # as post_norm reads the shapes
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    out = Guarded()
    es = 4 if dtype == torch.float32 else 2
    shift = es if off else 0
    new, new_t = out.empty((T, D), dtype, shift)
    h, h_t = out.empty((T, D), dtype, shift)
    ry, _ = out.empty((T,), torch.float32)
    rx, _ = out.empty((T,), torch.float32)
    head = (T, D, code(dtype), 0, code(gate_dtype), mode, 1, 0.7)
    rc = lib.gmm_sm100_post_norm(ptr(c["y"]), ptr(c["x"]), ptr(c["w"]), ptr(c["g"]), ptr(c["v"]), *head, 1e-6, 0.0, new, h,
                                 ry, rx, None)
    assert rc == 0, lib.gmm_sm100_last_error()
    dy, dy_t = out.empty((T, D), dtype, shift)
    dx, dx_t = out.empty((T, D), dtype, shift)
    dw, dw_t = out.empty((D,), torch.float32)
    dv, dv_t = out.empty((D,), torch.float32)
    dg, dg_t = out.empty(tuple(d["g"].shape), gate_dtype, shift if gate_dtype == dtype else 0) if mode else (None, None)
    size = lib.gmm_sm100_post_norm_backward_workspace_size(T, D)
    ws, _ = out.empty((size,), torch.uint8)
    rc = lib.gmm_sm100_post_norm_backward(ptr(c["y"]), ptr(c["x"]), ptr(c["w"]), ptr(c["g"]), ptr(c["v"]), ry, rx,
                                          ptr(c["dx"]), ptr(c["dh"]), *head, 0.0, dy, dx, dw, dg, dv, ws, size, None)
    assert rc == 0, lib.gmm_sm100_last_error()
    out.check()
    for k, t in (("new", new_t), ("h", h_t), ("dy", dy_t), ("dx", dx_t), ("dw", dw_t), ("dv", dv_t), ("dg", dg_t)):
        if t is None:
            continue
        if off:  # another layout adds in another order
            check(t(), formulas(d, "tanh", 0.7)[k], k)
        else:
            assert torch.equal(t(), want[k]), k
    # without a gradient of h: the next weight's gradient is left as it was
    before = dv_t()
    rc = lib.gmm_sm100_post_norm_backward(ptr(c["y"]), ptr(c["x"]), ptr(c["w"]), ptr(c["g"]), ptr(c["v"]), ry, rx,
                                          ptr(c["dx"]), None, *head, 0.0, dy, dx, dw, dg, None, ws, size, None)
    assert rc == 0, lib.gmm_sm100_last_error()
    out.check()
    assert torch.equal(dx_t(), c["dx"]) and torch.equal(dv_t(), before)
    check(dy_t(), formulas(d, "tanh", 0.7, use_dh=False)["dy"], "dy")
