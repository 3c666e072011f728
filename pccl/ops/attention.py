"""Attention for training: ``softmax(scale * q k^T) v`` and its gradients (``pccl/csrc/attention_fwd.cu``,
``attention_bwd.cu``).

The reference contains no attention (its DeepSpeed hook, ``pccl/patch_deepspeed.py:95-126``, expects an external GPT
training script); this is the attention of the GPT blocks (``pccl.models.gpt``, ``native_attention=True`` in the engine),
and it takes what those need beside it: shared key/value heads, queries and keys of different lengths (a chunk of a
sequence against the keys that the ranks have gathered so far), and documents packed one behind the other.

Layout.  ``q`` is ``[batch, rows, heads, dim]``, ``k`` and ``v`` are ``[batch, key rows, key heads, dim]``, bf16 or fp16;
``dim`` is a multiple of 8 up to 128 and ``heads`` a multiple of ``key heads`` (query head h reads key head
``h // (heads // key heads)``).  Only the last dimension has to be contiguous: views into a packed projection are read where
they lie (16-byte boundaries, strides that are multiples of 8 elements).  Packed sequences are ``[rows, heads, dim]`` with the
starts of the sequences and the end of the last one in ``cu_seqlens_q`` (and ``cu_seqlens_k``; left out, it is the same), int32
on the device, from 0 on and not decreasing; they are read there, so the host waits for nothing (starts that break this give
results that mean nothing, within the tensors).  Rows behind the last sequence belong to none: results that are allocated here
hold 0 there (``lse``: -inf), tensors given by the caller keep what they held.

Masks.  ``causal``: query i sees the keys up to ``i + (key rows - query rows)`` of its sequence, so that the last query sees the
last key.  A query that sees no key has an output of 0, an ``lse`` of -inf, and adds nothing to any gradient.
What is not finite in a hidden place (a value in the forward pass, any input in the backward pass) may make results of rows up
to 127 away from it NaN, because a probability of 0 is multiplied with it, as in the formula.  Nothing passes from one packed
sequence to another.

These are plain functions like those of ``pccl.ops.gemm``: they record nothing for autograd.  Results are the same bits from
call to call (no atomic additions).  Outputs must not overlap inputs or each other (views that lie in each other's range are
told apart where their strides are equal).  ``scale`` is positive.  Probabilities and score gradients are rounded to the
inputs' type for the products that they enter.  With fp16 that has a range: a score gradient above 65504 becomes infinite, as it does in
``dout``; below 6e-5 it loses digits and below 3e-8 it vanishes, so a loss whose gradients are small is scaled up first.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import build_kernels        # an import inside _C() would cost every call 0.6 us, of 7 for a small one


def _C():
    return build_kernels.load()


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True, scale: Optional[float] = None,
                      cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns ``(out, lse)``: the attention output in q's type and shape, and the logarithm of each query's sum of
    exponentials in fp32, ``[batch, heads, rows]`` (packed: ``[heads, rows]``), which the backward pass wants.
    ``scale`` is ``dim ** -0.5`` where it is not given."""
    return _C().attention_forward(q, k, v, causal, scale, cu_seqlens_q, cu_seqlens_k, out)


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                       causal: bool = True, scale: Optional[float] = None, cu_seqlens_q: Optional[torch.Tensor] = None,
                       cu_seqlens_k: Optional[torch.Tensor] = None, dq: Optional[torch.Tensor] = None,
                       dk: Optional[torch.Tensor] = None,
                       dv: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Returns ``(dq, dk, dv)`` for ``dout``, the gradient of the output; everything else is what the forward pass took and
    returned.  The probabilities are computed again from ``lse``.  The gradient of a shared key/value head is the sum over
    the query heads that read it.  ``dq``, ``dk`` and ``dv`` may be given, all three, and may be views into one packed gradient."""
    return _C().attention_backward(dout, q, k, v, out, lse, causal, scale, cu_seqlens_q, cu_seqlens_k, dq, dk, dv)


def check_errors(device: Optional[torch.device] = None) -> None:
    """Synchronise and raise if a bounded wait of an attention kernel on ``device`` has run out since the last check."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    torch.cuda.synchronize(idx)
    code = int(_C().attention_error(idx))
    if code != 0:
        _C().attention_reset_error(idx)
        raise RuntimeError(f"an attention kernel gave up in a bounded wait (code {code})")
