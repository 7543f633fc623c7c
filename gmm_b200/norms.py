"""The norms around a block, fused with its gate, its residual scale and its residual add.

A block ``f`` with RMS norms before and after it computes, for each row::

    h  = (v + o) * x  * r(x)                                   # pre_norm
    y  = f(h)
    x' = x + residual_scale * act(gate) * (w + o) * y * r(y)   # post_norm
    h' = (v' + o) * x' * r(x')                                 # the next block's pre-norm, in the same pass

with ``r(z) = 1 / sqrt(mean(z ** 2) + eps)`` over the last dimension and ``o``
the ``weight_offset``.  :func:`gmm_b200.moe.moe_block` runs an expert layer
between the two.  Both functions have gradients (one backward kernel); second
and forward-mode derivatives are refused.  A backward pass captured into a CUDA graph is refused
while a graph made on the default stream still holds one of the leaves given
here.  No reference counterpart.
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch

import gmm_b200

_GATE_ACTS = {"none": 0, "tanh": 1, "sigmoid": 2}


@functools.cache
def _op():
    if not gmm_b200._HAS_C:
        raise RuntimeError("gmm_b200._C is not available. Build with `python -m gmm_b200.build`.")
    return torch.ops.hopper_gmm_fwd.post_norm.default


def pre_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             weight_offset: float = 0.0) -> torch.Tensor:
    """RMS norm of ``x [..., dim]`` (CUDA, fp32/bf16/fp16, ``dim <= 16384``); ``weight [dim]`` of ``x``'s dtype or fp32."""
    return _op()(None, x, None, None, weight, 0, 1.0, eps, weight_offset, False)[1]


def post_norm(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
              gate: Optional[torch.Tensor] = None, gate_act: str = "none", residual_scale: float = 1.0,
              next_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              weight_offset: float = 0.0) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``residual + residual_scale * act(gate) * rms_norm(y)``, and the next block's pre-norm of it.

    Args:
        y, residual: ``[..., dim]`` CUDA, one dtype (fp32/bf16/fp16), ``dim <= 16384``.
        weight: ``[dim]`` post-norm weight, of their dtype or fp32.
        gate: ``[dim]`` (one a channel), ``[..., 1]`` (one a token) or
            ``[..., dim]``, of their dtype or fp32; ``None`` is 1.
        gate_act: ``"none"``, ``"tanh"`` or ``"sigmoid"``, applied to the gate.
        next_weight: ``[dim]`` weight of the next block's pre-norm (``weight``'s dtype).
        weight_offset: added to both weights (1 for weights stored around 0).

    Returns the new residual stream, and with ``next_weight`` also its norm
    (computed before the stream is rounded to its dtype).
    """
    if gate_act not in _GATE_ACTS:
        raise ValueError(f"gate_act must be one of {sorted(_GATE_ACTS)}, got {gate_act!r}")
    new, h, _ = _op()(y, residual, weight, gate, next_weight, _GATE_ACTS[gate_act], residual_scale, eps,
                        weight_offset, False)
    return new if next_weight is None else (new, h)
