"""A device-resident MoE expert layer built on the grouped GEMM.

``moe_forward(x, router_logits, w_gate_up, w_down, k)`` runs

1. top-k routing (softmax, k largest, optional renormalisation),
2. the permutation of the token rows into expert order (stable counting sort),
3. the fused SwiGLU gate/up grouped GEMM and the down grouped GEMM, both
   reading the per-expert row counts from device memory,
4. the weighted combine back into token order,

as seven kernel launches with no host synchronisation, so the layer can be
captured in a CUDA graph.  ``moe_forward_int8`` is the same layer on 8-bit
weights and activations, and ``moe_block`` puts the norms, the gate and the
residual around either.  The reference only provides step 3's grouped GEMM
(with host ``batch_sizes``); its benchmark leaves routing and gather/scatter
out (reference ``tests/bench_moe_forward.py:216-217``).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from gmm_b200 import capi
from gmm_b200.int8 import gmm_int8, gmm_int8_dev, quantize_rows
from gmm_b200.norms import post_norm


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _check_moe(rc):
    if rc != 0:
        raise RuntimeError(capi.load().gmm_sm100_moe_last_error().decode() or f"status {rc}")


def topk_route(logits: torch.Tensor, k: int, renormalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ids int32 [T, k], weights fp32 [T, k]) from router logits [T, E]."""
    if not logits.is_cuda or logits.dim() != 2:
        raise ValueError("logits must be a 2D CUDA tensor")
    logits = logits.contiguous()
    T, E = logits.shape
    ids = torch.empty(T, k, dtype=torch.int32, device=logits.device)
    w = torch.empty(T, k, dtype=torch.float32, device=logits.device)
    _check_moe(capi.load().gmm_sm100_moe_topk(logits.data_ptr(), capi.dtype_code(logits.dtype), T, E, k,
                                              int(renormalize), ids.data_ptr(), w.data_ptr(),
                                              _stream(logits)))
    return ids, w


def permute(x: Optional[torch.Tensor], ids: torch.Tensor, num_experts: int):
    """Token rows in expert order.

    Returns ``(x_perm [T*k, dim], batch_sizes int32 [E], dst_pos int32 [T, k],
    src_token int32 [T*k])``; all stay on the device.  With ``x = None`` only
    the positions are worked out and ``x_perm`` is ``None``."""
    if ids.dtype != torch.int32 or ids.dim() != 2 or not ids.is_cuda:
        raise ValueError("ids must be a 2D CUDA int32 tensor [T, k]")
    T, k = ids.shape
    dev = ids.device
    n = T * k
    x_perm, row_bytes = None, 0
    if x is not None:
        x = x.contiguous()
        if x.shape[0] != T:
            raise ValueError("x and ids must have the same number of tokens")
        x_perm = torch.empty(n, x.shape[1], dtype=x.dtype, device=x.device)
        row_bytes = x.shape[1] * x.element_size()
    bs = torch.empty(num_experts, dtype=torch.int32, device=dev)
    dst_pos = torch.empty(T, k, dtype=torch.int32, device=dev)
    src_token = torch.empty(n, dtype=torch.int32, device=dev)
    lib = capi.load()
    need = int(lib.gmm_sm100_moe_permute_workspace_size(n, num_experts))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    _check_moe(lib.gmm_sm100_moe_permute(None if x is None else x.data_ptr(), T, row_bytes,
                                         ids.contiguous().data_ptr(), k, num_experts,
                                         None if x is None else x_perm.data_ptr(),
                                         bs.data_ptr(), dst_pos.data_ptr(), src_token.data_ptr(),
                                         ws.data_ptr(), need, _stream(ids)))
    return x_perm, bs, dst_pos, src_token


def unpermute(y: torch.Tensor, dst_pos: torch.Tensor, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[dst_pos[t, j]]`` (fp32 accumulation)."""
    T, k = dst_pos.shape
    y = y.contiguous()
    out = torch.empty(T, y.shape[1], dtype=y.dtype, device=y.device)
    wp = weights.contiguous().float().data_ptr() if weights is not None else None
    _check_moe(capi.load().gmm_sm100_moe_unpermute(y.data_ptr(), dst_pos.contiguous().data_ptr(), wp, T, k,
                                                   y.shape[1], capi.dtype_code(y.dtype), out.data_ptr(),
                                                   _stream(y)))
    return out


def grouped_gemm_dev(a: torch.Tensor, b: torch.Tensor, batch_sizes: torch.Tensor,
                     trans_b: bool = False, swiglu: bool = False) -> torch.Tensor:
    """Grouped GEMM with device-resident int32 ``batch_sizes`` (no host sync).

    ``a`` has capacity rows; the first ``sum(batch_sizes)`` are used and only
    those rows of the result are written."""
    if batch_sizes.dtype != torch.int32 or not batch_sizes.is_cuda:
        raise ValueError("batch_sizes must be a CUDA int32 tensor")
    a = a.contiguous()
    b = b.contiguous()
    E = b.shape[0]
    dim_out = b.shape[1] if trans_b else b.shape[2]
    n_out = dim_out // 2 if swiglu else dim_out
    d = torch.empty(a.shape[0], n_out, dtype=a.dtype, device=a.device)
    dt = capi.dtype_code(a.dtype)
    lib = capi.load()
    need = int(lib.gmm_sm100_dev_workspace_size(E, a.shape[0], a.shape[1], dim_out, dt))
    ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
    capi._check(lib.gmm_sm100_forward_dev(a.data_ptr(), b.data_ptr(), batch_sizes.data_ptr(), E, a.shape[0],
                                          a.shape[1], dim_out, dt, int(trans_b), int(swiglu), d.data_ptr(),
                                          ws.data_ptr() if need else None, need, _stream(a)))
    return d


def moe_forward(x: torch.Tensor, router_logits: torch.Tensor, w_gate_up: torch.Tensor,
                w_down: torch.Tensor, k: int, trans_gate_up: bool = False, trans_down: bool = False,
                renormalize: bool = True) -> torch.Tensor:
    """MoE expert layer forward (SwiGLU experts) for tokens ``x [T, dim]``."""
    E = w_gate_up.shape[0]
    ids, w = topk_route(router_logits, k, renormalize)
    xp, bs, dst_pos, _ = permute(x, ids, E)
    h = grouped_gemm_dev(xp, w_gate_up, bs, trans_gate_up, swiglu=True)
    y = grouped_gemm_dev(h, w_down, bs, trans_down)
    return unpermute(y, dst_pos, w)


def moe_ffn_int8(a: torch.Tensor, w_gate_up: Tuple[torch.Tensor, torch.Tensor],
                 w_down: Tuple[torch.Tensor, torch.Tensor], batch_sizes: torch.Tensor) -> torch.Tensor:
    """``moe_ffn`` on 8-bit operands: expert-grouped rows ``a``, host ``batch_sizes``.

    The weights are ``quantize_experts`` pairs; activations are quantised row by
    row before each product, the hidden rows and the result have ``a``'s dtype
    (bf16 / fp16)."""
    q, scale = quantize_rows(a)
    h = gmm_int8(q, scale, *w_gate_up, batch_sizes, out_dtype=a.dtype, swiglu=True)
    q, scale = quantize_rows(h)
    return gmm_int8(q, scale, *w_down, batch_sizes, out_dtype=a.dtype)


def moe_forward_int8(x: torch.Tensor, router_logits: torch.Tensor, w_gate_up: Tuple[torch.Tensor, torch.Tensor],
                     w_down: Tuple[torch.Tensor, torch.Tensor], k: int, renormalize: bool = True) -> torch.Tensor:
    """``moe_forward`` on 8-bit operands (``quantize_experts`` pairs for the weights).

    Each token is quantised once, straight into the rows of its ``k`` experts;
    ``x`` is bf16 / fp16.  No host synchronisation."""
    E = w_gate_up[0].shape[0]
    ids, w = topk_route(router_logits, k, renormalize)
    _, bs, dst_pos, _ = permute(None, ids, E)
    q, scale = quantize_rows(x, dst_pos)
    h = gmm_int8_dev(q, scale, *w_gate_up, bs, out_dtype=x.dtype, swiglu=True)
    q, scale = quantize_rows(h)
    y = gmm_int8_dev(q, scale, *w_down, bs, out_dtype=x.dtype)
    return unpermute(y, dst_pos, w)


def _differentiated(t: torch.Tensor) -> bool:
    if t.requires_grad and torch.is_grad_enabled():
        return True
    # the level first: outside one, which is where a serving call is, unpacking ten arguments costs 18 us
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def moe_block(x: torch.Tensor, h: torch.Tensor, w_router: torch.Tensor, w_gate_up, w_down, k: int,
              post_weight: torch.Tensor, next_weight: Optional[torch.Tensor] = None,
              gate: Optional[torch.Tensor] = None, gate_act: str = "none", residual_scale: float = 1.0,
              eps: float = 1e-6, weight_offset: float = 0.0, renormalize: bool = True):
    """One MoE block of a serving model with norms around it.

    ``x [T, dim]`` is the residual stream and ``h`` its pre-norm (``pre_norm``
    for the first block, the second result of the previous ``moe_block``
    after that).  The router's logits are ``h @ w_router`` (``[dim, E]``); the
    expert weights are tensors (``moe_forward``) or ``quantize_experts`` pairs
    (``moe_forward_int8``).  Returns what :func:`gmm_b200.norms.post_norm` does:
    the new residual stream, and with ``next_weight`` the next block's ``h``.

    The expert layer has no backward pass, so an argument that requires a
    gradient (or carries a forward-mode one) is refused: run the block under
    ``torch.no_grad()``."""
    for t in (x, h, w_router, w_gate_up, w_down, post_weight, next_weight, gate):
        for part in (t,) if t is None or isinstance(t, torch.Tensor) else t:
            if part is not None and _differentiated(part):
                raise RuntimeError("moe_block has no backward pass through its expert layer, and an argument requires a "
                                   "gradient; run it under torch.no_grad()")
    layer = moe_forward if isinstance(w_gate_up, torch.Tensor) else moe_forward_int8
    y = layer(h, torch.matmul(h, w_router), w_gate_up, w_down, k, renormalize=renormalize)
    return post_norm(y, x, post_weight, gate=gate, gate_act=gate_act, residual_scale=residual_scale,
                     next_weight=next_weight, eps=eps, weight_offset=weight_offset)
