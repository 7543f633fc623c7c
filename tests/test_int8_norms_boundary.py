"""8-bit product, row quantiser and block norms without a GPU: host-side refusals of the C entry points (before any
CUDA call), op schemas and fake implementations."""

import numpy as np
import pytest
import torch

P = 4096  # a non-null, aligned dummy address; never dereferenced


def entry():
    from gmm_b200 import capi
    lib = capi.load()
    return lib, lambda: lib.gmm_sm100_last_error().decode()


def test_int8_entry_refuses_on_the_host():
    lib, last = entry()

    def call(bs=(3, 4), T=7, dim=32, dim_out=16, out=1, swiglu=0, a=P, sa=P, b=P, sb=P, d=P, ws=None):
        arr = np.asarray(bs, dtype=np.int64)
        return lib.gmm_sm100_forward_int8(a, sa, b, sb, arr.ctypes.data, len(bs), T, dim, dim_out, out, swiglu, d, ws, 0, None)

    assert call(T=8) == -2 and "Sum of batch_sizes (7)" in last()
    assert call(bs=(8, -1)) == -1 and "negative" in last()
    assert call(out=9) == -3
    assert call(dim=131072) == -8 and "131071" in last()
    assert call(out=0, swiglu=1) == -3
    assert call(dim_out=24, swiglu=1) == -4
    assert call(dim_out=12) == -4                      # 24-byte rows of D
    assert call(sa=None) == -1 and call(sb=None) == -1 and call(d=None) == -1
    assert call(sb=P + 8) == -4 and call(sa=P + 2) == -4 and call(d=P + 8) == -4
    assert call(bs=(0, 0), T=0) == 0                   # nothing to do


def test_int8_device_sizes_entry_refuses_on_the_host():
    lib, last = entry()

    def call(E=2, cap=8, dim=32, dim_out=16, out=1, swiglu=0, a=P, sa=P, b=P, sb=P, bs=P, d=P):
        return lib.gmm_sm100_forward_int8_dev(a, sa, b, sb, bs, E, cap, dim, dim_out, out, swiglu, d, None)

    assert call(E=0) == -1 and call(E=1025) == -1 and call(cap=-1) == -1
    assert call(out=5) == -3 and call(dim=131072) == -8 and call(out=0, swiglu=1) == -1
    assert call(sa=None) == -1 and call(sb=P + 4) == -4 and call(bs=P + 2) == -4 and call(bs=None) == -4
    assert call(d=P + 8) == -4 and call(dim_out=12) == -4
    assert call(cap=0) == 0


def test_int8_workspace_size():
    lib, _ = entry()
    few, many = np.ones(1024, dtype=np.int64), np.ones(1500, dtype=np.int64)
    assert lib.gmm_sm100_int8_workspace_size(few.ctypes.data, 1024, 1024, 32, 16) == 0
    assert lib.gmm_sm100_int8_workspace_size(many.ctypes.data, 1500, 1500, 32, 16) == ((3 * 1500 + 2) * 4 + 255) // 256 * 256
    assert lib.gmm_sm100_int8_workspace_size(many.ctypes.data, 1500, 3, 32, 16) == 0  # refused by the call itself


def test_quantize_rows_entry_refuses_on_the_host():
    lib, last = entry()

    def call(x=P, dtype=1, rows=4, dim=32, dst=None, k=1, out_rows=4, q=P, scale=P):
        return lib.gmm_sm100_quantize_rows(x, dtype, rows, dim, dst, k, out_rows, q, scale, None)

    assert call(rows=-1) == -1 and call(dim=-1) == -1 and call(out_rows=-1) == -1
    assert call(k=2) == -1 and call(dst=P, k=0) == -1 and call(dst=P, k=33) == -1
    assert call(out_rows=3) == -1 and "at least num_rows" in last()
    assert call(dtype=7) == -3
    assert call(dim=65537) == -8 and call(dst=P, rows=2 ** 31, out_rows=4) == -8
    assert call(x=None) == -1 and call(q=None) == -1 and call(scale=None) == -1
    assert call(q=P + 8) == -4 and call(x=P + 1) == -4 and call(scale=P + 2) == -4 and call(dst=P + 1) == -4
    assert call(rows=0, out_rows=0) == 0


def test_post_norm_entries_refuse_on_the_host():
    lib, last = entry()

    def fwd(y=P, x=P, w=P, g=None, v=P, rows=4, dim=32, dt=1, wdt=1, gdt=1, mode=0, act=0, eps=1e-6, xn=P, h=P):
        return lib.gmm_sm100_post_norm(y, x, w, g, v, rows, dim, dt, wdt, gdt, mode, act, 1.0, eps, 0.0, xn, h, None, None, None)

    assert fwd(rows=-1) == -1 and fwd(dim=-1) == -1 and fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1
    assert fwd(dt=4) == -3 and fwd(wdt=2) == -3 and fwd(gdt=2) == -3 and fwd(mode=4) == -1 and fwd(act=3) == -1
    assert fwd(dim=16385) == -8 and fwd(rows=2 ** 31) == -8
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(xn=None) == -1 and fwd(v=None) == -1
    assert fwd(y=None, h=None, v=None) == -1 and fwd(mode=1) == -1 and fwd(y=None, g=P, mode=1) == -1
    assert fwd(x=P + 1) == -4 and fwd(w=P + 2, wdt=0) == -4
    assert fwd(rows=0) == 0 and fwd(dim=0) == 0

    def bwd(y=P, x=P, w=P, g=None, v=P, ry=P, rx=P, dxn=P, dh=P, rows=4, dim=32, mode=0, dy=P, dx=P, dw=P, dg=None, dv=P):
        return lib.gmm_sm100_post_norm_backward(y, x, w, g, v, ry, rx, dxn, dh, rows, dim, 1, 1, 1, mode, 0, 1.0, 0.0, dy, dx, dw,
                                                dg, dv, None, 0, None)

    assert bwd(dxn=None, dh=None) == -1 and bwd(ry=None) == -1 and bwd(rx=None) == -1 and bwd(dy=None) == -1
    assert bwd(dx=None) == -1 and bwd(dw=None) == -1 and bwd(dv=None) == -1 and bwd(y=None, dh=None) == -1
    assert bwd(g=P, mode=1) == -1 and bwd(dim=16385) == -8 and bwd(ry=P + 2) == -4
    assert bwd(dim=0) == 0
    assert lib.gmm_sm100_post_norm_backward_workspace_size(0, 32) == 0
    assert lib.gmm_sm100_post_norm_backward_workspace_size(4, 20000) == 0


def test_schemas():
    import gmm_b200  # noqa: F401
    ops = torch.ops.hopper_gmm_fwd
    for name, schema in {
        "gmm_int8": "hopper_gmm_fwd::gmm_int8(Tensor A, Tensor a_scale, Tensor B, Tensor b_scale, Tensor batch_sizes, "
                    "ScalarType out_dtype, bool swiglu) -> Tensor",
        "quantize_rows": "hopper_gmm_fwd::quantize_rows(Tensor x, Tensor? dst_pos, SymInt out_rows) -> (Tensor, Tensor)",
    }.items():
        assert str(getattr(ops, name).default._schema).replace("SymInt", "int") == schema.replace("SymInt", "int")


def test_fake_impls():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from gmm_b200.int8 import gmm_int8, gmm_int8_dev, quantize_experts, quantize_rows
    from gmm_b200.norms import post_norm, pre_norm
    with FakeTensorMode():
        x = torch.empty(10, 40, dtype=torch.bfloat16, device="cuda")
        q, s = quantize_rows(x, torch.empty(10, 3, dtype=torch.int32, device="cuda"))
        assert q.shape == (30, 48) and q.dtype == torch.int8 and s.shape == (30,) and s.dtype == torch.float32
        wq, ws = quantize_experts(torch.empty(4, 40, 64, dtype=torch.bfloat16, device="cuda"))
        assert wq.shape == (4, 64, 48) and ws.shape == (4, 64)
        d = gmm_int8(q, s, wq, ws, torch.tensor([10, 0, 15, 5]), out_dtype=torch.float16)
        assert d.shape == (30, 64) and d.dtype == torch.float16 and d.device.type == "cuda"
        d = gmm_int8_dev(q, s, wq, ws, torch.empty(4, dtype=torch.int32, device="cuda"), swiglu=True)
        assert d.shape == (30, 32) and d.dtype == torch.bfloat16
        w = torch.empty(40, dtype=torch.bfloat16, device="cuda")
        new, h = post_norm(x, x, w, next_weight=w)
        assert new.shape == h.shape == x.shape and new.dtype == x.dtype
        assert pre_norm(x, w).shape == x.shape
        assert post_norm(x, x, w).shape == x.shape
        # a graph of fake tensors, and the backward operator's shapes (the engine itself needs a device)
        leaves = [t.requires_grad_() for t in (x, w, torch.empty(10, 1, dtype=torch.bfloat16, device="cuda"))]
        outs = post_norm(leaves[0], leaves[0], leaves[1], gate=leaves[2], next_weight=leaves[1])
        assert all(o.requires_grad for o in outs)
        stats = torch.empty(2, 10, dtype=torch.float32, device="cuda")
        with torch.no_grad():
            g = torch.ops.hopper_gmm_fwd.post_norm_backward(x, x, w, leaves[2], None, stats, outs[0], None, 0, 1.0, 0.0)
        assert [tuple(t.shape) for t in g] == [(10, 40), (10, 40), (40,), (10, 1), (0,)]


def test_cpu_tensors_have_no_kernel():
    from gmm_b200.int8 import quantize_rows
    from gmm_b200.norms import pre_norm
    with pytest.raises(NotImplementedError):
        quantize_rows(torch.zeros(2, 16))
    with pytest.raises(NotImplementedError):
        pre_norm(torch.zeros(2, 16), torch.zeros(16))
