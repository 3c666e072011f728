"""Norms of queries and keys for each head with the rotation of positions in the same pass (``pccl/csrc/rotary.cu``).

The reference contains no model (its DeepSpeed hook, ``pccl/patch_deepspeed.py:95-126``, expects an external GPT training
script); this is what the GPT blocks do between the QKV projection and attention when their configuration says
``qk_norm_rope=True``:

    n = x / sqrt(mean(x^2) + eps) * weight        over the columns of one head
    y = n, each pair (a, b) of its first ``rot`` columns turned: (a cos - b sin, b cos + a sin)

A pair is columns (i, i + rot / 2), or (2i, 2i + 1) with ``interleaved``; the rest of a head is not turned.

``q`` and ``k`` are ``[batch, rows, heads, dim]`` or ``[rows, heads, dim]``, bf16 or fp16, with a contiguous last dimension
of a multiple of 8 up to 256 (views into a packed projection are read where they lie: 16-byte boundaries, strides that are
multiples of 8 elements).  Weights are of that type or fp32.  ``cos`` and ``sin`` are fp32 tables, ``[positions, rot / 2]``
(``rotary_table``).  ``positions``, one for each row, int32 or int64 on the device, says where in the table a row stands;
without it that is the row's number.  A position that the table does not hold makes its row NaN.  An output may be exactly the
input that it comes from and overlaps nothing else of the call.  These are plain functions like those of ``pccl.ops.gemm``:
they record nothing for autograd.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import build_kernels        # an import inside _C() would cost every call 0.6 us, of 7 for a small one


def _C():
    return build_kernels.load()


def rotary_table(positions: int, rot: int, theta: float = 10000.0, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``cos`` and ``sin`` of ``position * theta ** (-2i / rot)``, computed in 64 bits (a far position times a frequency has no
    digits left behind the point in 32) and rounded once."""
    if rot < 8 or rot % 8 != 0:
        raise ValueError("rot must be a multiple of 8")
    freq = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def qk_norm_rope_forward(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                         sin: torch.Tensor, positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                         q_out: Optional[torch.Tensor] = None,
                         k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns the new ``(q, k)``; ``q_out`` and ``k_out`` may be given, and may be q and k themselves."""
    return _C().qk_norm_rope_forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, q_out, k_out)


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                          k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None,
                          eps: float = 1e-6, interleaved: bool = False, dq_in: Optional[torch.Tensor] = None,
                          dk_in: Optional[torch.Tensor] = None, dq_weight: Optional[torch.Tensor] = None,
                          dk_weight: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``dq`` and ``dk`` are the gradients of what the forward pass returned, ``q`` and ``k`` what it took.  Returns the
    gradients of ``q``, ``k`` (into ``dq_in`` and ``dk_in`` where given, which may be dq and dk themselves) and of the two
    weights (in their type; into ``dq_weight`` and ``dk_weight`` where given).  Results are the same bits from call to call."""
    return _C().qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, dq_in, dk_in, dq_weight,
                                      dk_weight)
