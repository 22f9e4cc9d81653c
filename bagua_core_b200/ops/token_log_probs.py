"""Log probabilities of given tokens, with entropy and the likeliest alternatives (`csrc/kernels/token_log_probs.h`).

    log_prob = x[target] - logsumexp(x)        entropy = -sum p log p

One pass over the logits forward, one backward; nothing of their size is kept in between, no probabilities and no fp32 copy.
A language model's loss is `-token_log_probs(logits, targets).log_probs.sum() / count`; policy gradients weigh the log
probabilities and add the entropy; a server returns the alternatives.

No counterpart in the reference, which has no model code."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .._native import C as _C

#: most alternatives of a row
MAX_TOP = _C.max_top_tokens


class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor                  # [...] fp32, differentiable
    entropy: torch.Tensor                    # [...] fp32, differentiable
    top_log_probs: Optional[torch.Tensor]    # [..., top] fp32, the likeliest first; not differentiable
    top_ids: Optional[torch.Tensor]          # [..., top] int64; of equal ones the lowest first


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, ignore_index: int = -100) -> TokenLogProbs:
    """logits [..., vocabulary] in float32, float16 or bfloat16, of any strides (rows whose elements are neighbours are read where they
    are); targets [...] of int64; `top`: how many alternatives, at most 32.

    A row whose target is `ignore_index` is not looked at: its log probability and entropy are 0, its gradient is 0, its
    alternatives are -inf with the id -1.  A row of nothing but -inf has the log probability -inf, the entropy 0 and
    no gradient; one with NaN or +inf gives NaN and the ids -1.  A target outside the vocabulary raises an error on the host; on a GPU its
    log probability is NaN, it has no gradient, and the next call raises the error."""
    return TokenLogProbs(*_C.token_log_probs(logits, targets, top, ignore_index))
