"""8-bit grouped product and row quantiser against integer and fp64 arithmetic.

Tolerances, as relative errors of a result from the exact value of its
definition (h = 2^-24, half a step of fp32):

* an integer sum below 2^31 rounds to fp32 once, and the two scales multiply it
  with one rounding each: 3 h, and half a step of the output type on top
  (bf16 2^-8, fp16 2^-11);
* SwiGLU with |gate| <= 16: the gate's own 3 h shift exp's argument by
  48 h, the fast exponential is within 2 + 1.173 * 16 < 21 steps (42 h), and
  the sum, quotient and two products add less than 8 h; the up value brings its
  3 h: below 128 h together;
* codes and scales are defined by correctly rounded fp32 divisions, which
  torch's CPU division is too, so they have to be equal.
"""

import pytest
import torch

import oracle
from gpu_util import forced_tile

pytestmark = pytest.mark.gpu

H = 2.0 ** -24
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# below the smallest normal fp16 the steps stop shrinking: half of 2^-24
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    from gmm_b200 import capi
    assert capi.device_error(clear=True) == 0


@pytest.fixture(params=["auto", "128", "256", "swap"])
def tile(request):
    with forced_tile(request.param):
        yield request.param


def problem(bs, dim, dim_out, seed=0):
    g = torch.Generator().manual_seed(seed)
    T, E = sum(bs), len(bs)
    a = torch.randint(-128, 128, (T, dim), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (E, dim_out, dim), generator=g, dtype=torch.int8)
    sa = torch.rand(T, generator=g) * 0.01 + 0.001
    sb = (torch.rand(E, dim_out, generator=g) * 0.01 + 0.001) / dim ** 0.5
    return a, sa, b, sb


def exact(a, sa, b, sb, bs, swiglu=False):
    """The definition in fp64 (every integer sum is below 2^53)."""
    out, at = [], 0
    for e, m in enumerate(bs):
        d = (a[at:at + m].double() @ b[e].double().t()) * sa[at:at + m].double()[:, None] * sb[e].double()
        at += m
        if swiglu:
            gate, up = d.chunk(2, dim=1)
            assert gate.numel() == 0 or gate.abs().max() <= 16
            d = gate / (1 + torch.exp(-gate)) * up
        out.append(d)
    return torch.cat(out)


def check(got, want, roundings):
    tol = want.abs() * (HALF_STEP[got.dtype] + roundings * H) * (1 + 2.0 ** -8) + TINY[got.dtype]
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double().cpu() - want).abs() / want.abs()).nan_to_num().max()))


def cuda(*ts):
    return [t.cuda() for t in ts]


RAGGED = [
    ([1], 16, 8),                                  # one token, the smallest contraction
    ([3, 0, 5, 1, 0], 48, 24),
    ([127, 128, 129, 1, 0, 255], 144, 264),        # around the tile height, columns past a tile
    ([0, 0, 257, 0], 1040, 520),
    ([400, 513, 385], 272, 520),                   # CTA-pair tiles with half-tile tails
    ([1] * 130 + [0] * 20, 80, 40),                # more groups than the small inline table
    ([16, 1, 0, 9, 15, 8], 2064, 48),              # decode: at most 16 rows an expert, the contraction split over warps
    ([2] * 100, 336, 328),                         # decode: more tasks than warps
]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,dim,dim_out", RAGGED)
def test_gmm_int8(bs, dim, dim_out, out, tile):
    from gmm_b200.int8 import gmm_int8, gmm_int8_dev
    p = problem(bs, dim, dim_out)
    d = cuda(*p)
    got = gmm_int8(*d, torch.tensor(bs), out_dtype=out)
    assert got.dtype == out and got.shape == (sum(bs), dim_out)
    check(got, exact(*p, bs), 3)
    dev = gmm_int8_dev(*d, torch.tensor(bs, dtype=torch.int32, device="cuda"), out_dtype=out)
    assert torch.equal(dev, got)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,dim,dim_out", [([1], 16, 16), ([127, 0, 130, 1], 208, 272), ([500, 390], 144, 528),
                                            ([1, 16, 0, 9], 2064, 96), ([5] * 90, 160, 336)])
def test_gmm_int8_swiglu(bs, dim, dim_out, out, tile):
    from gmm_b200.int8 import gmm_int8, gmm_int8_dev
    p = problem(bs, dim, dim_out, seed=1)
    d = cuda(*p)
    got = gmm_int8(*d, torch.tensor(bs), out_dtype=out, swiglu=True)
    assert got.shape == (sum(bs), dim_out // 2)
    check(got, exact(*p, bs, swiglu=True), 128)
    dev = gmm_int8_dev(*d, torch.tensor(bs, dtype=torch.int32, device="cuda"), out_dtype=out, swiglu=True)
    assert torch.equal(dev, got)


@pytest.mark.parametrize("bs", [[3, 0, 2], [300, 500]])
def test_gmm_int8_largest_sums(bs, tile):
    """Codes of -128 everywhere at the largest contraction: the sum is 128 * 128 * 131056, just below 2^31."""
    from gmm_b200.int8 import gmm_int8
    dim, dim_out = 131056, 8
    a = torch.full((sum(bs), dim), -128, dtype=torch.int8, device="cuda")
    b = torch.full((len(bs), dim_out, dim), -128, dtype=torch.int8, device="cuda")
    b[:, 1] = 127  # the most negative sum beside it
    got = gmm_int8(a, torch.ones(sum(bs), device="cuda"), b, torch.ones(len(bs), dim_out, device="cuda"),
                   torch.tensor(bs), out_dtype=torch.float32)
    want = torch.full((sum(bs), dim_out), float(128 * 128 * dim))
    want[:, 1] = -128.0 * 127 * dim
    assert torch.equal(got.cpu(), want.float())


def test_gmm_int8_many_experts_use_the_workspace_table():
    from gmm_b200.int8 import gmm_int8
    bs = [1, 2] * 600
    p = problem(bs, 32, 16, seed=2)
    check(gmm_int8(*cuda(*p), torch.tensor(bs), out_dtype=torch.float32), exact(*p, bs), 3)


def test_gmm_int8_special_scales_and_padding():
    """A zero scale gives zeros, a NaN scale NaN in its row or column only, an infinite one infinities;
    rows behind the last expert's stay as they were."""
    from gmm_b200.int8 import gmm_int8_dev
    bs = [5, 130, 0, 7]
    a, sa, b, sb = problem(bs, 64, 72, seed=3)
    sa[2] = 0.0
    sa[9] = float("nan")
    sb[1, 30] = float("inf")
    b[1, 30] = 1
    a[10] = 1  # a positive sum under the infinite scale
    spare = 40
    a2 = torch.cat([a, torch.full((spare, 64), 77, dtype=torch.int8)])
    sa2 = torch.cat([sa, torch.full((spare,), float("nan"))])
    A, SA, B, SB = cuda(a2, sa2, b, sb)
    lib_out = torch.full((sum(bs) + spare, 72), -3.0, dtype=torch.float32, device="cuda")
    from gmm_b200 import capi
    sizes = torch.tensor(bs, dtype=torch.int32, device="cuda")
    capi._check(capi.load().gmm_sm100_forward_int8_dev(
        A.data_ptr(), SA.data_ptr(), B.data_ptr(), SB.data_ptr(), sizes.data_ptr(), 4, A.shape[0], 64, 72,
        capi.GMM_DTYPE_F32, 0, lib_out.data_ptr(), torch.cuda.current_stream().cuda_stream))
    got = gmm_int8_dev(A, SA, B, SB, sizes, out_dtype=torch.float32)
    out = lib_out.cpu()
    assert torch.equal(got[:sum(bs)].cpu().nan_to_num(5.0), out[:sum(bs)].nan_to_num(5.0))
    assert (out[sum(bs):] == -3.0).all()
    assert (out[2] == 0).all() and out[9].isnan().all() and out[10, 30] == float("inf")
    keep = [r for r in range(sum(bs)) if r not in (2, 9)]
    cols = [c for c in range(72) if c != 30]
    want = exact(a, sa, b, sb, bs)
    check(out[keep][:, cols], want[keep][:, cols], 3)


@pytest.mark.parametrize("bs", [[], [0, 0]])
def test_gmm_int8_without_rows(bs):
    from gmm_b200.int8 import gmm_int8
    a, sa, b, sb = problem(bs, 32, 16)
    got = gmm_int8(*cuda(a, sa, b, sb), torch.tensor(bs, dtype=torch.int64))
    assert got.shape == (0, 16)


def test_gmm_int8_empty_contraction_is_zero():
    from gmm_b200.int8 import gmm_int8
    got = gmm_int8(torch.empty(5, 0, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"),
                   torch.empty(2, 16, 0, dtype=torch.int8, device="cuda"), torch.ones(2, 16, device="cuda"),
                   torch.tensor([2, 3]))
    assert (got == 0).all()


def test_gmm_int8_refusals():
    from gmm_b200.int8 import gmm_int8, gmm_int8_dev
    a, sa, b, sb = cuda(*problem([3, 4], 32, 16))
    bs = torch.tensor([3, 4])
    for args, text in [((a.float(), sa, b, sb, bs), "int8"), ((a, sa[:-1], b, sb, bs), "a_scale"),
                       ((a, sa, b, sb.t(), bs), "b_scale"), ((a, sa, b, sb.double(), bs), "b_scale"),
                       ((a[:, :16].contiguous(), sa, b, sb, bs), r"B.size\(2\)"), ((a, sa, b, sb, bs[:1]), r"B.size\(0\)"),
                       ((a, sa, b, sb, torch.tensor([3, 3])), "Sum of batch_sizes"),
                       ((a, sa, b, sb, torch.tensor([8, -1])), "negative"),
                       ((a[:, ::2], sa, b, sb, bs), "contiguous"),
                       ((a[:, :24].contiguous(), sa, b[:, :, :24].contiguous(), sb, bs), "multiple of 16"),
                       ((a, sa, b, sb, bs.int()), "CPU int64")]:
        with pytest.raises(RuntimeError, match=text):
            gmm_int8(*args)
    with pytest.raises(RuntimeError, match="bf16 / fp16"):
        gmm_int8(a, sa, b, sb, bs, out_dtype=torch.float32, swiglu=True)
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        gmm_int8(a, sa, b, sb, bs, out_dtype=torch.int32)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        gmm_int8(a, sa, b[:, :12].contiguous(), sb[:, :12].contiguous(), bs)  # 24-byte rows of D
    with pytest.raises(RuntimeError, match="CUDA int32"):
        gmm_int8_dev(a, sa, b, sb, bs)
    with pytest.raises(RuntimeError, match="131071"):
        gmm_int8(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), sa[:1],
                 torch.zeros(1, 8, 131072, dtype=torch.int8, device="cuda"), sb[:1, :8].contiguous(), torch.tensor([1]))


def test_bad_device_sizes_are_recorded_not_followed():
    from gmm_b200 import capi
    from gmm_b200.int8 import gmm_int8_dev
    a, sa, b, sb = cuda(*problem([60, 40], 32, 16))
    for sizes, status in (([80, 30], -2), ([-1, 30], -1), ([2 ** 31 - 1, 2 ** 31 - 1], -2)):
        gmm_int8_dev(a, sa, b, sb, torch.tensor(sizes, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert capi.device_error(clear=True) == status


# ------------------------------------------------------------------ quantiser
def spec_quantize(x):
    """The definition with torch's CPU fp32 divisions (tensor by tensor: correctly rounded)."""
    f = x.float()
    top = f.abs().amax(dim=1) if x.shape[1] else torch.zeros(x.shape[0])
    scale = top / torch.full_like(top, 127.0)
    scale[~torch.isfinite(f).all(dim=1)] = float("nan")
    ok = scale > 0
    q = torch.round(f / torch.where(ok, scale, 1.0)[:, None]).clamp(-127, 127)
    q[~ok] = 0
    width = (x.shape[1] + 15) // 16 * 16
    return torch.nn.functional.pad(q, (0, width - x.shape[1])).to(torch.int8), scale


def rows_of(T, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, dim, generator=g) * torch.logspace(-3, 2, T)[:, None]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,dim", [(1, 1), (1, 8), (3, 16), (5, 100), (9, 2048), (4, 2050), (3, 2057), (7, 4096), (2, 16384),
                                   (2, 16392), (1, 30001), (1, 65536)])
def test_quantize_rows(T, dim, dtype):
    from gmm_b200.int8 import quantize_rows
    x = rows_of(T, dim, dtype)
    q, scale = quantize_rows(x.cuda())
    want_q, want_scale = spec_quantize(x)
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(q.cpu(), want_q)
    # what the codes stand for, in fp64: within half a code (and the division's rounding, 127 h)
    back = q[:, :dim].double().cpu() * want_scale.double()[:, None]
    assert ((back - x.double()).abs() <= want_scale.double()[:, None] * (0.5 + 128 * H)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_quantize_rows_next_to_halves(dtype):
    """Values at, and one step of fp32 around, every half-way point between two codes, for several scales."""
    from gmm_b200.int8 import quantize_rows
    halves = torch.arange(-127, 127).float() + 0.5
    rows = []
    for top in (127.0, 1.0, 126.99999, 3.3e-30, 0.7, 2.0 ** -118, 2.0 ** -130):
        scale = torch.tensor(top) / torch.tensor(127.0)
        mid = halves * scale
        for v in (mid, torch.nextafter(mid, torch.tensor(float("inf"))), torch.nextafter(mid, torch.tensor(float("-inf")))):
            rows.append(torch.cat([torch.tensor([top]), v]))
    x = torch.stack(rows).to(dtype)
    x = x[torch.isfinite(x).all(1)]
    q, scale = quantize_rows(x.cuda())
    want_q, want_scale = spec_quantize(x)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu(), want_q)


def test_quantize_rows_unaligned_and_strided():
    from gmm_b200.int8 import quantize_rows
    base = rows_of(13, 520, torch.bfloat16, seed=4).cuda()
    for x in (base[:, 3:515], base[::2], base.t(), base.reshape(-1)[1:1 + 5 * 1024].view(5, 1024)):
        q, scale = quantize_rows(x)
        want_q, want_scale = spec_quantize(x.cpu())
        assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu(), want_q)


def test_quantize_rows_special_rows():
    from gmm_b200.int8 import quantize_rows
    x = rows_of(9, 40, torch.float32, seed=5)
    x[0] = 0.0
    x[1, 7] = float("inf")
    x[2, 39] = float("nan")
    x[3] = 0.0
    x[3, 1] = 1e-44          # a scale that rounds to zero
    x[4] = 0.0
    x[4, :3] = torch.tensor([3.4e38, -3.4e38, 1.3e36])  # the largest values
    x[5] = 0.0
    x[5, 5] = 190 * 2.0 ** -149  # its scale is one denormal step: the code is held at 127
    x[6] = -x[6].abs()
    x[7, 0] = float("-inf")
    x[7, 1] = float("nan")
    q, scale = quantize_rows(x.cuda())
    want_q, want_scale = spec_quantize(x)
    assert torch.equal(scale.cpu().isnan(), want_scale.isnan()) and scale.cpu()[[1, 2, 7]].isnan().all()
    assert torch.equal(scale.cpu().nan_to_num(9.0), want_scale.nan_to_num(9.0))
    assert torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("T,k,dim", [(1, 1, 16), (6, 3, 50), (33, 8, 256), (5, 32, 24)])
def test_quantize_rows_into_places(T, k, dim):
    from gmm_b200.int8 import quantize_rows
    x = rows_of(T, dim, torch.float16, seed=6)
    g = torch.Generator().manual_seed(7)
    place = torch.randperm(T * k, generator=g).view(T, k).to(torch.int32)
    q, scale = quantize_rows(x.cuda(), place.cuda())
    want_q, want_scale = spec_quantize(x)
    src = torch.empty(T * k, dtype=torch.long)
    src[place.long().reshape(-1)] = torch.arange(T).repeat_interleave(k)
    assert torch.equal(q.cpu(), want_q[src]) and torch.equal(scale.cpu(), want_scale[src])


def test_quantize_rows_skips_places_outside():
    """Positions outside the result (an id outside the experts gives -1) are skipped; unnamed rows stay as they were."""
    from gmm_b200 import capi
    x = rows_of(3, 32, torch.bfloat16, seed=8).cuda()
    place = torch.tensor([[0, -1], [6, 3], [2 ** 31 - 1, 4]], dtype=torch.int32, device="cuda")
    q = torch.full((7, 32), 55, dtype=torch.int8, device="cuda")
    scale = torch.full((7,), -1.0, device="cuda")
    capi._check(capi.load().gmm_sm100_quantize_rows(x.data_ptr(), capi.GMM_DTYPE_BF16, 3, 32, place.data_ptr(), 2, 7,
                                                    q.data_ptr(), scale.data_ptr(),
                                                    torch.cuda.current_stream().cuda_stream))
    want_q, want_scale = spec_quantize(x.cpu())
    for row, src in {0: 0, 6: 1, 3: 1, 4: 2}.items():
        assert torch.equal(q[row].cpu(), want_q[src]) and scale[row].cpu() == want_scale[src]
    for row in (1, 2, 5):
        assert (q[row] == 55).all() and scale[row] == -1.0


def test_quantize_rows_refusals_and_empty():
    from gmm_b200.int8 import quantize_experts, quantize_rows
    x = torch.randn(4, 32, device="cuda")
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        quantize_rows(x.double())
    with pytest.raises(RuntimeError, match="2D"):
        quantize_rows(x[0], out_rows=1)
    with pytest.raises(RuntimeError, match="int32"):
        quantize_rows(x, torch.zeros(4, 2, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="num_rows, k"):
        quantize_rows(x, torch.zeros(3, 2, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="k <= 32"):
        quantize_rows(x, torch.zeros(4, 33, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="at least num_rows"):
        quantize_rows(x, out_rows=3)
    with pytest.raises(RuntimeError, match="65536"):
        quantize_rows(torch.zeros(1, 65537, device="cuda"))
    with pytest.raises(RuntimeError, match="3D"):
        quantize_experts(x)
    q, s = quantize_rows(torch.empty(0, 20, device="cuda"))
    assert q.shape == (0, 32) and s.shape == (0,)
    q, s = quantize_rows(torch.empty(3, 0, device="cuda"))
    assert q.shape == (3, 0) and (s == 0).all()


@pytest.mark.parametrize("trans_b", [False, True])
def test_quantize_experts(trans_b):
    from gmm_b200.int8 import quantize_experts
    g = torch.Generator().manual_seed(9)
    w = torch.randn(3, 20, 24, generator=g).bfloat16()
    q, s = quantize_experts(w.cuda(), trans_b)
    rows = w if trans_b else w.transpose(1, 2)
    want_q, want_s = spec_quantize(rows.reshape(-1, rows.shape[2]))
    assert q.shape == (3, rows.shape[1], 32) and torch.equal(q.cpu().view(-1, 32), want_q)
    assert torch.equal(s.cpu().view(-1), want_s)


# ------------------------------------------------------------------ together
def layer(T=600, E=16, k=2, dim=256, inter=320, seed=4, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, dim, generator=g).to(dtype)
    logits = torch.randn(T, E, generator=g)
    w1 = (torch.randn(E, dim, 2 * inter, generator=g) / dim ** 0.5).to(dtype)
    w2 = (torch.randn(E, inter, dim, generator=g) / inter ** 0.5).to(dtype)
    return x, logits, w1, w2


@pytest.mark.parametrize("T", [1, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_forward_int8(T, dtype, tile):
    """Against the layer in fp64.  A code is off by a uniform half step: s / sqrt(12) with s = max / 127, and the
    largest of 256..320 normal values is below 4.2 sigma, so an operand's relative error is below 0.0096, a product's
    (two operands) 0.0136.  SwiGLU adds the errors of gate and up (its slope in the gate is below 1.1 of its own size
    on average): 0.0212; the second product: (0.0212^2 + 0.0136^2)^1/2 = 0.026, and the 16-bit roundings 0.004."""
    from gmm_b200.int8 import quantize_experts
    from gmm_b200.moe import moe_forward_int8
    x, logits, w1, w2 = layer(T=T, dtype=dtype)
    q1, q2 = quantize_experts(w1.cuda()), quantize_experts(w2.cuda())
    got = moe_forward_int8(x.cuda(), logits.cuda(), q1, q2, k=2).double().cpu()
    ids, w = oracle.topk_oracle(logits, 2)
    want = torch.zeros_like(got)
    for j in range(2):
        e = torch.from_numpy(ids[:, j]).long()
        gu = torch.bmm(x.double()[:, None], w1.double()[e])[:, 0]
        gate, up = gu.chunk(2, dim=1)
        y = torch.bmm((gate * torch.sigmoid(gate) * up)[:, None], w2.double()[e])[:, 0]
        want += torch.from_numpy(w[:, j]).double()[:, None] * y
    # a single token has few values to average over: twice the allowance
    assert (got - want).norm() <= (0.030 if T > 1 else 0.060) * want.norm()


def test_moe_forward_int8_is_its_parts_and_ffn_agrees():
    from gmm_b200.int8 import gmm_int8_dev, quantize_experts, quantize_rows
    from gmm_b200.moe import moe_ffn_int8, moe_forward_int8, permute, topk_route, unpermute
    x, logits, w1, w2 = (t.cuda() for t in layer())
    q1, q2 = quantize_experts(w1), quantize_experts(w2)
    got = moe_forward_int8(x, logits, q1, q2, k=2)
    ids, w = topk_route(logits, 2)
    xp, bs, dst, _ = permute(x, ids, 16)
    a, sa = quantize_rows(xp)  # gathered first, quantised after: the same rows
    h = gmm_int8_dev(a, sa, *q1, bs, swiglu=True)
    y = gmm_int8_dev(*quantize_rows(h), *q2, bs)
    assert torch.equal(got, unpermute(y, dst, w))
    assert torch.equal(moe_ffn_int8(xp, q1, q2, bs.cpu().long()), y)


def test_layer_without_tokens():
    from gmm_b200.int8 import quantize_experts
    from gmm_b200.moe import moe_forward_int8
    x, logits, w1, w2 = (t.cuda() for t in layer(T=4))
    q1, q2 = quantize_experts(w1), quantize_experts(w2)
    out = moe_forward_int8(x[:0], logits[:0], q1, q2, k=2)
    assert out.shape == (0, 256) and out.dtype == x.dtype


def test_every_token_to_one_expert(tile):
    """Device sizes chosen as for few rows an expert, all of them on one."""
    from gmm_b200.int8 import gmm_int8_dev
    bs = [0] * 40 + [500] + [0] * 23
    p = problem(bs, 96, 48, seed=12)
    got = gmm_int8_dev(*cuda(*p), torch.tensor(bs, dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    check(got, exact(*p, bs), 3)


def test_concurrent_host_threads():
    """Calls from four host threads on streams of their own, with different kernels each."""
    import threading
    from gmm_b200.int8 import gmm_int8, quantize_rows
    jobs = [problem(bs, 272, 136, seed=20 + i) + (bs,) for i, bs in enumerate(([3, 1, 9], [200, 0, 70], [900, 500], [16] * 30))]
    want = [exact(*j[:4], j[4]) for j in jobs]
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            d = cuda(*jobs[i][:4])
            x = rows_of(50 + i, 400, torch.bfloat16, seed=i)
            for _ in range(20):
                got = gmm_int8(*d, torch.tensor(jobs[i][4]), out_dtype=torch.float32)
                q, s = quantize_rows(x.cuda())
                torch.cuda.current_stream().synchronize()
                wq, ws = spec_quantize(x)
                if not (torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)):
                    wrong.append(("quantize", i))
                if ((got.double().cpu() - want[i]).abs() > want[i].abs() * 4 * H).any():
                    wrong.append(("gmm", i))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_permute_without_rows():
    from gmm_b200.moe import permute
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 7, (50, 3), generator=g, dtype=torch.int32).cuda()
    x = torch.randn(50, 16, device="cuda")
    full, bare = permute(x, ids, 7), permute(None, ids, 7)
    assert bare[0] is None and all(torch.equal(a, b) for a, b in zip(full[1:], bare[1:]))


def test_layer_captured_twice_and_on_two_streams():
    """Two graphs of the layer with different inputs, replayed in turn and at once on two streams."""
    from gmm_b200.int8 import quantize_experts
    from gmm_b200.moe import moe_forward_int8
    x, logits, w1, w2 = (t.cuda() for t in layer())
    x2, logits2, _, _ = (t.cuda() for t in layer(seed=11))
    q1, q2 = quantize_experts(w1), quantize_experts(w2)
    eager = [moe_forward_int8(x, logits, q1, q2, k=2), moe_forward_int8(x2, logits2, q1, q2, k=2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a, l in ((x, logits), (x2, logits2)):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            moe_forward_int8(a, l, q1, q2, k=2)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = moe_forward_int8(a, l, q1, q2, k=2)
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
    # new tokens through the first graph
    x.copy_(x2)
    logits.copy_(logits2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager[1])


def test_large_table_is_not_captured():
    from gmm_b200.int8 import gmm_int8
    bs = torch.ones(1100, dtype=torch.int64)
    a, sa, b, sb = cuda(*problem([1] * 1100, 16, 8))
    want = gmm_int8(a, sa, b, sb, bs)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="captured"):
                gmm_int8(a, sa, b, sb, bs)
        finally:
            graph.capture_end()
    torch.cuda.synchronize()
    assert torch.equal(gmm_int8(a, sa, b, sb, bs), want)


def test_rows_past_32_bit_offsets():
    """A [T, dim] whose last rows lie beyond 2^31 elements: quantised and multiplied like any other."""
    from gmm_b200.int8 import gmm_int8, quantize_rows
    T, dim = 70_000, 32_768
    x = torch.zeros(T, dim, dtype=torch.float16, device="cuda")
    g = torch.Generator().manual_seed(3)
    tail = torch.randn(5, dim, generator=g).half()
    x[-5:] = tail.cuda()
    q, scale = quantize_rows(x)
    want_q, want_s = spec_quantize(tail)
    assert torch.equal(q[-5:].cpu(), want_q) and torch.equal(scale[-5:].cpu(), want_s)
    b = torch.randint(-128, 128, (1, 8, dim), generator=g, dtype=torch.int8)
    sb = torch.ones(1, 8)
    got = gmm_int8(q, scale, b.cuda(), sb.cuda(), torch.tensor([T]), out_dtype=torch.float32)
    check(got[-5:], exact(want_q, want_s, b, sb, [5]), 3)
    assert (got[:-5] == 0).all()


def test_weights_past_32_bit_offsets(tile):
    """The last of 140 experts lies beyond 2^31 bytes of weights."""
    from gmm_b200.int8 import gmm_int8
    experts, dim = 140, 4096
    bs = [2] + [0] * (experts - 2) + [5]
    a, sa, last, s_last = problem([7], dim, dim)
    b = torch.zeros(experts, dim, dim, dtype=torch.int8, device="cuda")
    sb = torch.ones(experts, dim, device="cuda")
    b[-1], sb[-1] = last[0].cuda(), s_last[0].cuda()
    got = gmm_int8(a.cuda(), sa.cuda(), b, sb, torch.tensor(bs), out_dtype=torch.float32)
    assert (got[:2] == 0).all()
    check(got[2:], exact(a[2:], sa[2:], last, s_last, [5]), 3)
