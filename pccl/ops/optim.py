"""AdamW over a list of tensors in one launch, with states in 32 or in 8 bits (``pccl/csrc/adamw_multi.cu``).

The reference has no optimizer (DeepSpeed brings its own, ``pccl/patch_deepspeed.py:95-126``).  ``pccl._C.adamw`` steps one
flat shard; this steps every tensor of a list, with a weight decay for each, and can keep both moments in 8 bits: 2 bytes
and 2/64 of a byte of scales per parameter instead of 8 (``optim_bits=8`` in the ZeRO-3 engine).

The states of a list are flat: each tensor's part starts on a multiple of 256 elements, in the order of the list.  With 8
bits, 256 elements share a scale, and a value between two codes is rounded to one of them by chance so that its mean is
kept; the chance is a function of ``seed``, ``step`` and the element's place, so the same call gives the same bits.
Second moments of a block that are all below 2^-80 are held as zeros, so with 8 bits ``eps`` has to be large enough
(``least_eps``) that their roots do not count beside it.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .. import build_kernels        # an import inside _C() would cost every call 0.6 us, of 7 for a small one

BLOCK = 256


def _C():
    return build_kernels.load()


def least_eps(beta2: float) -> float:
    """The smallest ``eps`` that 8-bit states take: 2^-35 / sqrt(1 - beta2), 1.3e-10 at 0.95, 9.2e-10 at 0.999.  The update of an
    element whose second moment is held as zero is then too large by 1/32 of itself at most."""
    return _C().adamw_least_eps(beta2)


def state_offsets(params: Sequence[torch.Tensor]) -> List[int]:
    """Where each tensor's part of the flat states begins, and where the last one ends."""
    at = [0]
    for p in params:
        at.append(at[-1] + (p.numel() + BLOCK - 1) // BLOCK * BLOCK)
    return at


@dataclass
class AdamWState:
    """First and second moments: fp32, or int8 and uint8 codes with an fp32 scale for each block of 256."""

    exp_avg: torch.Tensor
    exp_avg_sq: torch.Tensor
    exp_avg_scale: Optional[torch.Tensor] = None
    exp_avg_sq_scale: Optional[torch.Tensor] = None

    @property
    def bits(self) -> int:
        return 32 if self.exp_avg_scale is None else 8

    def dequantize(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Both moments as flat fp32 tensors: the states themselves where they are fp32, else new ones."""
        if self.exp_avg_scale is None:
            return self.exp_avg, self.exp_avg_sq
        return _C().adamw_dequantize(self.exp_avg, self.exp_avg_sq, self.exp_avg_scale, self.exp_avg_sq_scale)


def adamw_state(params: Sequence[torch.Tensor], bits: int = 32) -> AdamWState:
    """Zero moments for ``params``."""
    if bits not in (8, 32):
        raise ValueError("bits must be 8 or 32")
    if len(params) == 0:
        raise ValueError("adamw_state needs at least one parameter")
    n, dev = state_offsets(params)[-1], params[0].device
    if bits == 32:
        return AdamWState(torch.zeros(n, dtype=torch.float32, device=dev), torch.zeros(n, dtype=torch.float32, device=dev))
    return AdamWState(torch.zeros(n, dtype=torch.int8, device=dev), torch.zeros(n, dtype=torch.uint8, device=dev),
                      torch.zeros(n // BLOCK, dtype=torch.float32, device=dev), torch.zeros(n // BLOCK, dtype=torch.float32, device=dev))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], state: AdamWState, *, step: int, lr: float,
               beta1: float = 0.9, beta2: float = 0.95, eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 0.1,
               masters: Optional[Sequence[torch.Tensor]] = None, grad_scale: float = 1.0, max_grad_norm: float = 0.0,
               total_sq_norm: Optional[torch.Tensor] = None, seed: int = 0) -> None:
    """One step, in place, of every tensor in ``params``: bf16 or fp16 with an fp32 ``master`` each, which the step updates and
    rounds into the parameter, or fp32 without.  Gradients are bf16, fp16 or fp32.  All parameters have one dtype, all
    gradients one; every tensor is contiguous, and none that the step writes may overlap another.

    ``step`` counts from 1.  ``weight_decay`` is one number, or one for each tensor.  Gradients are multiplied by
    ``grad_scale``, and with ``max_grad_norm`` > 0 scaled down where their norm, ``sqrt(total_sq_norm) * grad_scale``, is above
    it; ``total_sq_norm`` is a device scalar (``pccl._C.sq_norm`` adds to one, ranks may add theirs), read on the device.  All other
    numbers are the call's own: a captured call replays with the ``step``, ``lr`` and noise that it was captured with."""
    decay = [float(weight_decay)] if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
    _C().adamw_multi(list(params), list(grads), None if masters is None else list(masters), state.exp_avg, state.exp_avg_sq,
                     state.exp_avg_scale, state.exp_avg_sq_scale, decay, step, lr, beta1, beta2, eps, grad_scale, max_grad_norm,
                     total_sq_norm, seed)
