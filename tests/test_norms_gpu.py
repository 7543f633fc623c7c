"""Norms around a block, forward and backward, against their formulas in fp64.

Tolerances follow the computation: a result that is a chain of fp32 operations
is within K * 2^-24 of its formula with every term taken by its absolute value
(the running error bound).  K counts the roundings along the longest chain: a
row sum adds at most 8 * 4 terms in a thread and 10 levels across the block
(42), the mean, eps and reciprocal root 7, a gate's tanh or sigmoid and its slope 18
(the fast exponential 2 |g| + 4 with |g| < 4.5, the sum, the reciprocal, the slope's
product), and the products, the norm they multiply and the second sum less than 60 more:
K = 128.  Sums over rows add one rounding a row.  Cancellation in
x' = x + P enlarges what r(x') carries by |x| + |P| over |x'|, by norm; that
factor multiplies K.  Half a step of the output type comes on top.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

H = 2.0 ** -24
K = 128
HALF_STEP = {torch.float32: H, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -130, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


def inputs(T, D, dtype, params=None, gate="none", following=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    params = params or dtype
    d = {"y": torch.randn(T, D, generator=g).to(dtype), "x": (torch.randn(T, D, generator=g) * 1.5).to(dtype),
         "w": (torch.rand(D, generator=g) + 0.5).to(params),
         "v": (torch.rand(D, generator=g) - 0.7).to(params) if following else None,
         "dx": torch.randn(T, D, generator=g).to(dtype),
         "dh": torch.randn(T, D, generator=g).to(dtype) if following else None}
    shape = {"none": None, "channel": (D,), "token": (T, 1), "full": (T, D)}[gate]
    d["g"] = None if shape is None else torch.randn(shape, generator=g).to(params if gate == "channel" else dtype)
    return d


def act(g, kind):
    if g is None:
        one = torch.ones((), dtype=torch.float64)
        return one, 0 * one
    if kind == "tanh":
        a = torch.tanh(g)
        return a, 1 - a * a
    if kind == "sigmoid":
        a = torch.sigmoid(g)
        return a, a * (1 - a)
    return g, torch.ones_like(g)


def f64(d, k):
    return None if d[k] is None else d[k].detach().double().cpu()


def formulas(d, kind="none", s=1.0, eps=1e-6, o=0.0, use_dx=True, use_dh=True):
    """{name: (value, bound / (K 2^-24))} of the outputs and gradients, all in fp64."""
    y, x, w, v, g, dxn, dh = (f64(d, k) for k in ("y", "x", "w", "v", "g", "dx", "dh"))
    D = x.shape[1]
    ry = (y.square().mean(1, keepdim=True) + eps).rsqrt()
    yh = y * ry
    a, da = act(g, kind)
    P = s * a * (w + o) * yh
    new = x + P
    mag = x.abs() + P.abs()
    res = {"new": (new, mag)}
    dx = dxn if use_dx else torch.zeros_like(x)
    m_dx = dx.abs()
    if v is not None:
        rx = (new.square().mean(1, keepdim=True) + eps).rsqrt()
        kappa = 1 + mag.norm(dim=1, keepdim=True) / new.norm(dim=1, keepdim=True).clamp_min(1e-30)
        res["h"] = ((v + o) * new * rx, (v + o).abs() * rx * mag * kappa)
        if use_dh:
            xh, m_xh = new * rx, mag * rx * kappa
            u = dh * (v + o)
            dx = dx + rx * (u - xh * (u * xh).mean(1, keepdim=True))
            m_dx = m_dx + rx * kappa * (u.abs() + m_xh * (u.abs() * m_xh).mean(1, keepdim=True))
            res["dv"] = ((dh * xh).sum(0), (dh.abs() * m_xh).sum(0) * (1 + x.shape[0] / K))
    q = s * a * (w + o)
    t, m_t = q * dx, q.abs() * m_dx
    res["dx"] = (dx, m_dx)
    res["dy"] = (ry * (t - yh * (t * yh).mean(1, keepdim=True)),
                 ry * (m_t + yh.abs() * (m_t * yh.abs()).mean(1, keepdim=True)))
    rows = 1 + x.shape[0] / K
    res["dw"] = ((s * a * dx * yh).sum(0), ((s * a).abs() * m_dx * yh.abs()).sum(0) * rows)
    if g is not None:
        dg = s * (w + o) * yh * dx * da
        # the slope of a saturated gate comes from 1 - a^2 or a (1 - a): bounded by a itself, not by the slope
        m_dg = abs(s) * ((w + o) * yh).abs() * m_dx * torch.maximum(da.abs(), torch.ones_like(da) * 1.0)
        how = "full" if g.shape == x.shape else "channel" if g.dim() == 1 else "token"
        res["dg"] = {"full": (dg, m_dg), "channel": (dg.sum(0), m_dg.sum(0) * rows),
                     "token": (dg.sum(1, keepdim=True), m_dg.sum(1, keepdim=True))}[how]
    return res


def check(got, want, what):
    value, bound = want
    tol = value.abs() * HALF_STEP[got.dtype] * (1 + 2.0 ** -8) + K * H * bound + TINY[got.dtype]
    off = (got.detach().double().cpu() - value).abs()
    assert (off <= tol).all(), (what, float((off / tol).max()))


def cuda(d):
    return {k: None if t is None else t.cuda() for k, t in d.items()}


def forward(c, kind="none", s=1.0, eps=1e-6, o=0.0):
    from gmm_b200.norms import post_norm
    return post_norm(c["y"], c["x"], c["w"], gate=c["g"], gate_act=kind, residual_scale=s, next_weight=c["v"], eps=eps,
                     weight_offset=o)


def train(c, kind="none", s=1.0, eps=1e-6, o=0.0, use_dx=True, use_dh=True):
    names = [k for k in ("y", "x", "w", "v", "g") if c[k] is not None]
    leaves = {k: c[k].detach().clone().requires_grad_() for k in names}
    out = forward({**c, **leaves}, kind, s, eps, o)
    new, h = out if c["v"] is not None else (out, None)
    outs = [(t, gr) for t, gr, use in ((new, c["dx"], use_dx), (h, c["dh"], use_dh)) if t is not None and use]
    grads = torch.autograd.grad([t for t, _ in outs], list(leaves.values()), [gr for _, gr in outs], allow_unused=True)
    res = {"d" + k: gr for k, gr in zip(names, grads)}
    res["new"] = new
    if h is not None:
        res["h"] = h
    return res


SIZES = [(1, 1), (40, 1), (1, 8), (3, 7), (700, 3), (2000, 18), (5, 33), (4, 64), (9, 250), (7, 256), (300, 264), (5, 2048), (3, 2050), (2, 4096),
         (3, 5000), (2, 6144), (3, 8200), (2, 16384)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", SIZES)
def test_sizes_forward_and_backward(T, D, dtype):
    d = inputs(T, D, dtype, gate="channel")
    want = formulas(d, "none", 0.7)
    got = train(cuda(d), "none", 0.7)
    for k in ("new", "h", "dy", "dx", "dw", "dv", "dg"):
        check(got[k], want[k], k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(5, 64), (400, 33), (3, 4096), (9, 2050)])
def test_rows_off_the_16_byte_grid(T, D, dtype):
    """Every tensor starts one to three elements into its buffer, and the buffers end with the last row."""
    d = inputs(T, D, dtype, gate="full", seed=21)
    want = formulas(d, "sigmoid", 0.7)
    c = {}
    for i, (k, t) in enumerate(d.items()):
        buf = torch.empty(t.numel() + 1 + i % 3, dtype=t.dtype, device="cuda")
        c[k] = buf[1 + i % 3:].view(t.shape)
        c[k].copy_(t)
    leaves = {k: c[k].requires_grad_() for k in ("y", "x", "w", "v", "g")}
    new, h = forward(c, "sigmoid", 0.7)
    grads = torch.autograd.grad((new, h), list(leaves.values()), (c["dx"], c["dh"]))
    check(new, want["new"], "new")
    check(h, want["h"], "h")
    for k, gr in zip(leaves, grads):
        check(gr, want["d" + k], k)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("kind", ["none", "tanh", "sigmoid"])
@pytest.mark.parametrize("dtype,params", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float32, torch.float32)])
@pytest.mark.parametrize("D", [72, 75])
def test_gates(gate, kind, dtype, params, D):
    for following in (True, False):
        d = inputs(37, D, dtype, params, gate, following, seed=2)
        want = formulas(d, kind, -0.3, eps=1e-5, o=1.0)
        c = cuda(d)
        got = train(c, kind, -0.3, 1e-5, 1.0)
        for k, v in got.items():
            check(v, want[k], (k, following))
        out = forward(c, kind, -0.3, 1e-5, 1.0)  # without a graph: the same values
        for a, b in zip(out if following else (out,), (got["new"], got.get("h"))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("gate", ["token", "full"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", [(21, 64), (700, 77), (1500, 250), (33, 4091), (19, 5003)])
def test_fp32_gate_beside_16_bit_rows(T, D, dtype, gate):
    d = inputs(T, D, dtype, dtype, gate, seed=22)
    d["g"] = d["g"].float() * 1.01
    want = formulas(d, "sigmoid", 0.6)
    got = train(cuda(d), "sigmoid", 0.6)
    assert got["dg"].dtype == torch.float32
    for k, v in got.items():
        check(v, want[k], k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(3000, 1), (3000, 9), (2500, 31), (1200, 255), (700, 1026), (450, 4083), (330, 8190)])
def test_many_rows_off_the_word(T, D, dtype):
    """Rows that start anywhere in a 16-byte word, several to a block; nothing is written outside the outputs."""
    d = inputs(T, D, dtype, torch.float32, "channel", seed=23)
    want = formulas(d, "tanh", 0.7)
    got = train(cuda(d), "tanh", 0.7)
    for k, v in got.items():
        check(v, want[k], k)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype,params", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("T,D", [(1, 8193), (200, 8200), (170, 16383), (160, 16384), (9, 12288)])
def test_wide_rows(T, D, dtype, params, gate):
    """Backward in column windows: each row's sums are put together from the windows'."""
    d = inputs(T, D, dtype, params, gate, seed=24)
    want = formulas(d, "sigmoid", 0.6)
    got = train(cuda(d), "sigmoid", 0.6)
    for k, v in got.items():
        check(v, want[k], k)


@pytest.mark.parametrize("use_dx,use_dh", [(True, False), (False, True)])
@pytest.mark.parametrize("gate", ["none", "token"])
def test_one_output_used(use_dx, use_dh, gate):
    d = inputs(20, 104, torch.bfloat16, torch.float32, gate, seed=3)
    want = formulas(d, "tanh", 0.5, use_dx=use_dx, use_dh=use_dh)
    got = train(cuda(d), "tanh", 0.5, use_dx=use_dx, use_dh=use_dh)
    for k in ("dy", "dx", "dw") + (("dg",) if gate == "token" else ()):
        check(got[k], want[k], k)
    if use_dh:
        check(got["dv"], want["dv"], "dv")
    else:
        assert (got["dv"] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(1, 16), (21, 100), (260, 4096)])
def test_pre_norm(T, D, dtype):
    from gmm_b200.norms import pre_norm
    d = inputs(T, D, dtype, torch.float32, seed=4)
    d["y"] = torch.zeros_like(d["y"])  # P = 0: the formulas' x' is x
    want = formulas(d, o=1.0, use_dx=False)
    x, v = d["x"].cuda().requires_grad_(), d["v"].cuda().requires_grad_()
    h = pre_norm(x, v, weight_offset=1.0)
    dx, dv = torch.autograd.grad(h, (x, v), d["dh"].cuda())
    check(h, want["h"], "h")
    check(dx, want["dx"], "dx")
    check(dv, want["dv"], "dv")
    with torch.no_grad():
        assert torch.equal(pre_norm(x, v, weight_offset=1.0), h)


@pytest.mark.parametrize("gate,kind", [("none", "none"), ("channel", "tanh"), ("token", "sigmoid"), ("full", "tanh")])
def test_gradients_against_differences(gate, kind):
    """The directional derivative of the fp64 definition by central differences of step e = 1e-4 (truncation e^2 times a
    third derivative of order one, 1e-8 against values of order one) against the kernel's fp32 gradients, whose error is
    within K * 2^-24 < 1e-5 of their magnitudes: 1e-4 of the sum of magnitudes covers both."""
    d = inputs(6, 24, torch.float32, gate=gate, seed=5)
    got = train(cuda(d), kind, 0.8, 1e-5, 0.5)

    def loss(moved):
        m = {**d, **moved}
        r = formulas(m, kind, 0.8, 1e-5, 0.5)
        return float((r["new"][0] * d["dx"].double()).sum() + (r["h"][0] * d["dh"].double()).sum())

    g = torch.Generator().manual_seed(6)
    for k in ("y", "x", "w", "v", "g"):
        if d[k] is None:
            continue
        way = torch.randn(d[k].shape, generator=g, dtype=torch.float64)
        e = 1e-4
        diff = (loss({k: d[k].double() + e * way}) - loss({k: d[k].double() - e * way})) / (2 * e)
        grad = got["d" + k].double().cpu() * way
        assert abs(float(grad.sum()) - diff) <= 1e-4 * float(grad.abs().sum()) + 1e-6, k


def test_special_values_stay_in_their_rows():
    """Zero rows are zeros through both norms; an infinity or NaN spoils its own row only, forward and backward
    (the sums over rows carry it, as their formula does)."""
    d = inputs(6, 40, torch.float32, gate="full", seed=7)
    d["y"][0] = 0
    d["x"][1] = 0
    d["y"][1] = 0
    d["y"][2, 3] = float("nan")
    d["x"][3, 5] = float("inf")
    clean = [0, 1, 4, 5]
    c = cuda(d)
    got = train(c, "tanh", 0.5)
    sub = {k: t if t is None or t.shape[0] == 40 else t[clean] for k, t in d.items()}
    want = formulas(sub, "tanh", 0.5)
    for k in ("new", "h", "dx", "dy", "dg"):
        check(got[k][clean], want[k], k)
    assert (got["h"][1] == 0).all()
    assert got["new"][2].isnan().all() and got["h"][2].isnan().all()
    assert got["dw"].isnan().any()


def test_shapes_strides_and_broadcasts():
    from gmm_b200.norms import post_norm, pre_norm
    g = torch.Generator().manual_seed(8)
    big = torch.randn(4, 6, 200, generator=g).cuda()
    y, x = big[:, :5, 3:163], big.transpose(0, 1)[:5, :, 20:180].transpose(0, 1)  # [4, 5, 160], strided
    w, v = torch.rand(320, generator=g).cuda()[::2], torch.rand(160, generator=g).cuda()
    gate = torch.randn(4, 5, 1, generator=g).cuda()
    new, h = post_norm(y, x, w, gate=gate, next_weight=v)
    flat = post_norm(y.reshape(20, 160), x.reshape(20, 160), w.contiguous(), gate=gate.reshape(20, 1), next_weight=v)
    assert new.shape == h.shape == (4, 5, 160)
    assert torch.equal(new.view(20, 160), flat[0]) and torch.equal(h.view(20, 160), flat[1])
    # an expanded gate: the gradient is summed back over what it was shared by
    shared = torch.randn(4, 1, 160, generator=g).cuda().requires_grad_()
    out = post_norm(y, x, w, gate=shared.expand(4, 5, 160), gate_act="sigmoid")
    (ds,) = torch.autograd.grad(out, shared, big[:, :5, :160])
    d = {"y": y.reshape(20, 160), "x": x.reshape(20, 160), "w": w, "v": None, "dh": None,
         "dx": big[:, :5, :160].reshape(20, 160), "g": shared.expand(4, 5, 160).reshape(20, 160)}
    value, bound = formulas(d, "sigmoid")["dg"]
    check(ds, (value.view(4, 5, 160).sum(1, keepdim=True), bound.view(4, 5, 160).sum(1, keepdim=True)), "shared gate")
    # one row without batch dimensions, and none at all
    one = pre_norm(x[0, 0], v)
    assert torch.equal(one, pre_norm(x[0, :1].contiguous(), v)[0])
    empty = post_norm(y[:0], x[:0], w, next_weight=v)
    assert empty[0].shape == empty[1].shape == (0, 5, 160)


def test_gradients_of_no_rows_are_zero():
    from gmm_b200.norms import post_norm
    y = torch.empty(0, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    v = torch.ones(32, device="cuda", requires_grad=True)
    gate = torch.ones(32, device="cuda", requires_grad=True)
    new, h = post_norm(y, y, w, gate=gate, next_weight=v)
    grads = torch.autograd.grad((new, h), (w, v, gate), (new.detach(), h.detach()))
    assert all((t == 0).all() and t.shape == (32,) for t in grads)


def test_same_leaf_twice_and_inputs_unchanged():
    """y and the residual may be one tensor, weights one parameter; nothing is written in place."""
    from gmm_b200.norms import post_norm
    d = inputs(11, 48, torch.float32, seed=9)
    x, w = d["x"].cuda().requires_grad_(), d["w"].cuda().requires_grad_()
    before = x.detach().clone()
    new, h = post_norm(x, x, w, next_weight=w)
    dx, dw = torch.autograd.grad((new, h), (x, w), (d["dx"].cuda(), d["dh"].cuda()))
    r = formulas({**d, "y": d["x"], "v": d["w"], "g": None})
    check(dx, (r["dx"][0] + r["dy"][0], r["dx"][1] + r["dy"][1]), "dx")
    check(dw, (r["dw"][0] + r["dv"][0], r["dw"][1] + r["dv"][1]), "dw")
    assert torch.equal(x.detach(), before)


def test_results_do_not_change_from_run_to_run():
    c = cuda(inputs(3001, 1024, torch.bfloat16, torch.float32, "channel", seed=10))
    first = train(c, "tanh")
    for _ in range(3):
        again = train(c, "tanh")
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_refusals():
    from gmm_b200.norms import post_norm, pre_norm
    x = torch.randn(4, 32, device="cuda")
    w = torch.ones(32, device="cuda")
    for kw, text in [(dict(gate=torch.ones(5, device="cuda")), "gate must have shape"),
                     (dict(gate=torch.ones(4, 32, device="cuda").half()), "rows' dtype or be fp32"),
                     (dict(next_weight=torch.ones(31, device="cuda")), r"\[dim\]"),
                     (dict(next_weight=torch.ones(32)), "rows' device"),
                     (dict(eps=-1.0), "eps")]:
        with pytest.raises(RuntimeError, match=text):
            post_norm(x, x, w, **kw)
    with pytest.raises(RuntimeError, match="same shape and dtype"):
        post_norm(x.half(), x, w)
    with pytest.raises(RuntimeError, match="same shape and dtype"):
        post_norm(x[:2], x, w)
    with pytest.raises(RuntimeError, match="one dtype"):
        post_norm(x.half(), x.half(), w.half(), next_weight=w)
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        pre_norm(x.double(), w)
    with pytest.raises(RuntimeError, match="16384"):
        pre_norm(torch.zeros(1, 16385, device="cuda"), torch.zeros(16385, device="cuda"))
    with pytest.raises(ValueError, match="gate_act"):
        post_norm(x, x, w, gate_act="relu")
    x = x.requires_grad_()
    out = post_norm(x, x, w)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), x, create_graph=True)


def test_captured_forward_and_backward():
    """A step captured into a graph (fresh leaves, no eager graph of them alive) and replayed on new values."""
    d = cuda(inputs(130, 264, torch.bfloat16, torch.float32, "channel", seed=12))
    want = train(d, "tanh")
    d2 = cuda(inputs(130, 264, torch.bfloat16, torch.float32, "channel", seed=13))
    want2 = train(d2, "tanh")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        train(d, "tanh")
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train(d, "tanh")
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out[k], want[k]) for k in want)
    for k, t in d.items():
        if t is not None:
            t.copy_(d2[k])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out[k], want2[k]) for k in want2)


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    from gmm_b200.norms import post_norm
    x, y, w = (torch.randn(*shape, device="cuda").requires_grad_() for shape in ((5, 16), (5, 16), (16,)))
    alive = post_norm(y, x, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still holds an input"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(post_norm(y, x, w)[0].sum(), (x, y, w))
    torch.cuda.synchronize()
    # the eager graph is intact, and once it is gone the same step is captured
    want = torch.autograd.grad(alive[0].sum(), (x, y, w))
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(post_norm(y, x, w)[0].sum(), (x, y, w))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    cs = [cuda(inputs(700, 1000, torch.bfloat16, torch.float32, "full", seed=20 + i)) for i in range(2)]
    want = [train(c, "sigmoid") for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(train(c, "sigmoid"))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[k], b[k]) for k in b)


def test_rows_past_32_bit_offsets():
    from gmm_b200.norms import post_norm
    T, D = 140_000, 16_384
    y = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    d = inputs(3, D, torch.bfloat16, seed=14)
    y[-3:] = d["y"].cuda()
    new, h = post_norm(y, y, d["w"].cuda(), next_weight=d["v"].cuda())
    want = formulas({**d, "x": d["y"], "g": None})
    check(new[-3:], want["new"], "new")
    check(h[-3:], want["h"], "h")
    assert (new[:-3] == 0).all()


@pytest.mark.parametrize("int8", [False, True])
def test_moe_block(int8):
    """Two blocks in a row are the calls they are made of."""
    from gmm_b200.int8 import quantize_experts
    from gmm_b200.moe import moe_block, moe_forward, moe_forward_int8
    from gmm_b200.norms import post_norm, pre_norm
    g = torch.Generator().manual_seed(15)
    T, dim, inter, E, k = 70, 128, 96, 8, 2
    x = torch.randn(T, dim, generator=g).bfloat16().cuda()
    norms = [(torch.rand(dim, generator=g) + 0.5).bfloat16().cuda() for _ in range(4)]
    gate = torch.randn(dim, generator=g).bfloat16().cuda()
    layers = []
    for _ in range(2):
        router = (torch.randn(dim, E, generator=g) / dim ** 0.5).bfloat16().cuda()
        w1 = (torch.randn(E, dim, 2 * inter, generator=g) / dim ** 0.5).bfloat16().cuda()
        w2 = (torch.randn(E, inter, dim, generator=g) / inter ** 0.5).bfloat16().cuda()
        layers.append((router, quantize_experts(w1) if int8 else w1, quantize_experts(w2) if int8 else w2))
    h = pre_norm(x, norms[0])
    x1, h1 = moe_block(x, h, *layers[0], k, norms[1], next_weight=norms[2], gate=gate, gate_act="tanh", residual_scale=0.5)
    x2 = moe_block(x1, h1, *layers[1], k, norms[3])
    run = moe_forward_int8 if int8 else moe_forward
    y = run(h, h @ layers[0][0], layers[0][1], layers[0][2], k)
    want1, want_h1 = post_norm(y, x, norms[1], gate=gate, gate_act="tanh", residual_scale=0.5, next_weight=norms[2])
    y = run(want_h1, want_h1 @ layers[1][0], layers[1][1], layers[1][2], k)
    assert torch.equal(x1, want1) and torch.equal(h1, want_h1) and torch.equal(x2, post_norm(y, want1, norms[3]))
