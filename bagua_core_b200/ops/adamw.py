"""AdamW over many tensors in one launch, with its moments in fp32 or in 8 bits (`csrc/kernels/adamw.h`).

    m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g²
    p = p (1 - lr wd) - lr / (1 - b1^t) · m / (sqrt(v / (1 - b2^t)) + eps)

`bagua_core_b200.parallel.FlatAdamW` is the optimizer built on it.

Moments in 8 bits take 2 bytes a parameter instead of 8, and a step moves 16 bytes instead of 28.  256 neighbouring
elements of a tensor share an fp32 scale for each moment; a code is a small floating point number (first moment: sign, 4
bits of exponent, 3 of fraction; second: 4 and 4).  Rounding is stochastic, so that moments which change by less than
a code's distance in one step still follow their mean; its random bits are a hash of seed, step, tensor and element, so
that a step can be repeated bit for bit.  A second moment above zero stays above zero.

No counterpart in the reference, which has no optimizer."""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from .._native import C as _C

#: elements of a tensor that share the scales of its 8-bit moments
MOMENT8_BLOCK = _C.moment8_block


def adamw_state8(p: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes of the first moment, codes of the second, scales [2, blocks]) of a tensor's 8-bit moments, all zero."""
    blocks = (p.numel() + MOMENT8_BLOCK - 1) // MOMENT8_BLOCK
    codes = [torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format, requires_grad=False) for _ in range(2)]
    return codes[0], codes[1], torch.zeros(2, blocks, dtype=torch.float32, device=p.device)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], *, step: Union[int, torch.Tensor], lr: float, betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, scales: Optional[Sequence[torch.Tensor]] = None,
               copies: Optional[Sequence[torch.Tensor]] = None, seed: int = 0, first_index: int = 0, stream=None) -> int:
    """Steps all `params` (lists or tuples of tensors) in place and returns how many kernels that took.

    Parameters are float32, float16 or bfloat16, gradients of their type or float32, or of any of the three where the
    parameters are float32; the arithmetic is fp32.  Each tensor has its elements without gaps, and its gradient, its moments
    and its copy have its sizes and strides.  All tensors of a call are on one device (a GPU or the host) and of one kind.
    Moments are float32, or, with `scales`, uint8 codes as `adamw_state8` makes them.  `copies`: bfloat16 tensors that
    receive the new parameters.  `step`: the number of this step, from 1; or one int64 on the parameters' device, read when the
    step runs, which is what a captured step needs.  `seed`: of the rounding of 8-bit moments; `first_index`: the first
    tensor's number among all those that are stepped with one seed."""
    if stream is not None and params and params[0].is_cuda:
        with torch.cuda.stream(stream):
            return _C.adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales, copies, lr, betas[0], betas[1], eps, weight_decay, step,
                                 seed, first_index)
    return _C.adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales, copies, lr, betas[0], betas[1], eps, weight_decay, step, seed,
                         first_index)


def adamw_read8(exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], scales: Sequence[torch.Tensor],
                exp_avgs_out: Sequence[torch.Tensor], exp_avg_sqs_out: Sequence[torch.Tensor], stream=None) -> int:
    """Writes the values that 8-bit moments stand for into tensors of float32, float16 or bfloat16 and of the codes' sizes and
    strides; returns how many kernels that took."""
    if stream is not None and exp_avgs and exp_avgs[0].is_cuda:
        with torch.cuda.stream(stream):
            return _C.adamw_read8(exp_avgs, exp_avg_sqs, scales, exp_avgs_out, exp_avg_sqs_out)
    return _C.adamw_read8(exp_avgs, exp_avg_sqs, scales, exp_avgs_out, exp_avg_sqs_out)
