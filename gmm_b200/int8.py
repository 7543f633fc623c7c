"""8-bit (W8A8) grouped products: int8 rows and weights, one scale a token and one a channel.

``quantize_experts`` lays the weights out once; a call then quantises its
activations (``quantize_rows``) and multiplies (``gmm_int8``, or
``gmm_int8_dev`` with device-resident batch sizes)::

    wq, ws = quantize_experts(w)                       # once, at load time
    aq, as_ = quantize_rows(a)                         # int8 codes, fp32 scale per row
    d = gmm_int8(aq, as_, wq, ws, batch_sizes)         # d[rows_e] ~ a[rows_e] @ w[e]

Sums are exact 32-bit integers; the scaled result is fp32, rounded once to
``out_dtype``.  A weight pair ``(wq, ws)`` also goes where :mod:`gmm_b200.moe`
takes expert weights (``moe_ffn_int8``, ``moe_forward_int8``).  These are
serving operators: no gradient flows through them.  No reference counterpart
(the reference multiplies fp32 / bf16 / fp16 only).
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

import gmm_b200


@functools.cache
def _op(name: str):
    if not gmm_b200._HAS_C:
        raise RuntimeError("gmm_b200._C is not available. Build with `python -m gmm_b200.build`.")
    return getattr(torch.ops.hopper_gmm_fwd, name).default


def quantize_rows(x: torch.Tensor, dst_pos: Optional[torch.Tensor] = None,
                  out_rows: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``x [T, dim]`` (CUDA, fp32/bf16/fp16) as 8-bit codes and a scale each.

    ``scale = max|x| / 127`` and ``code = rint(x / scale)`` (both divisions
    correctly rounded in fp32), so ``x ~ code * scale``.  Returns ``(codes int8
    [R, dim rounded up to 16], scale fp32 [R])``; the columns past ``dim`` are
    zero and add nothing to a product.

    With ``dst_pos`` (int32 ``[T, k]``, ``k <= 32``; the one
    :func:`gmm_b200.moe.permute` returns) row ``t`` is written to the rows
    ``dst_pos[t, j]`` of the result, ``R = out_rows`` (default ``T * k``);
    positions outside ``[0, R)`` are skipped and rows nobody names are left
    unwritten.  A row of zeros has scale 0; a row that holds an infinity or a
    NaN has scale NaN, which makes every product with it NaN.
    """
    if out_rows is None:
        out_rows = x.shape[0] * (1 if dst_pos is None else dst_pos.shape[1])
    return _op("quantize_rows")(x, dst_pos, out_rows)


def quantize_experts(w: torch.Tensor, trans_b: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Expert weights for :func:`gmm_int8`: int8 codes and one scale for each output channel.

    ``w`` is ``[E, dim, dim_out]``, or ``[E, dim_out, dim]`` with ``trans_b``
    (the layouts of ``hopper_gmm_fwd``; ``[gate | up]`` side by side for SwiGLU
    as in ``gmm_swiglu``).  Returns ``(codes int8 [E, dim_out, dim rounded up to
    16], scale fp32 [E, dim_out])``.  Run once, when weights are loaded.
    """
    if w.dim() != 3:
        raise RuntimeError("w must be 3D [num_experts, dim, dim_out] (or [num_experts, dim_out, dim])")
    rows = w if trans_b else w.transpose(1, 2)
    E, n, dim = rows.shape
    with torch.no_grad():  # of parameters too: the scales are data, not a function of them
        q, scale = quantize_rows(rows.reshape(E * n, dim))
    return q.view(E, n, q.shape[1]), scale.view(E, n)


def gmm_int8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
             batch_sizes: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
             swiglu: bool = False) -> torch.Tensor:
    """8-bit grouped GEMM: ``out[i, n] = a_scale[i] * b_scale[e, n] * sum_k a[i, k] * b[e, n, k]``.

    Args:
        a: ``[num_tokens, dim]`` contiguous CUDA int8, ``dim`` a multiple of 16
           (``quantize_rows`` pads to it) and at most 131071.
        a_scale: ``[num_tokens]`` fp32.
        b: ``[num_experts, dim_out, dim]`` contiguous CUDA int8 (``quantize_experts``).
        b_scale: ``[num_experts, dim_out]`` fp32.
        batch_sizes: ``[num_experts]`` int64 tensor on CPU, as in ``hopper_gmm_fwd``.
        out_dtype: bf16, fp16 or fp32; ``dim_out`` times its size must be a
           multiple of 16 bytes.
        swiglu: ``b`` holds ``[gate rows | up rows]``; returns
           ``silu(gate) * up`` of the scaled sums, ``[num_tokens, dim_out // 2]``
           (bf16 / fp16, ``dim_out`` a multiple of 16).
    """
    return _op("gmm_int8")(a, a_scale, b, b_scale, batch_sizes, out_dtype, swiglu)


def gmm_int8_dev(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                 batch_sizes: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
                 swiglu: bool = False) -> torch.Tensor:
    """:func:`gmm_int8` with device-resident int32 ``batch_sizes`` (no host sync, at most 1024 experts).

    ``a`` has capacity rows; the first ``sum(batch_sizes)`` are used and only
    those rows of the result are written."""
    return _op("gmm_int8_dev")(a, a_scale, b, b_scale, batch_sizes, out_dtype, swiglu)
