"""Rows of a table looked up by token and scaled, for any number of tokens (`csrc/kernels/embedding.h`).

    out[t] = scale · table[ids[t]]        dtable[v] = scale · sum of dout[t] over the tokens t with ids[t] = v

The gradient goes by sorted tokens: one stable sort of the ids, then one pass over the gradient of the output, which writes each
row of the table's gradient once, in the tokens' order.  Sums are fp32 and rounded once; the same call gives the same bits.

No counterpart in the reference, which has no model code."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .._native import C as _C
from . import wgrad as _wgrad


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """`scale * table[ids]` in `dtype` (the table's by default), one rounding from fp32.

    ids: int64 or int32 of any shape; table: [rows, columns] in float32, float16 or bfloat16, on the ids' device; `padding_idx`
    names a row that gets no gradient (negative: counted from the end).  An id outside the table raises an error on the host; on a GPU it
    gives a row of NaN, takes no part in the gradient, and the next call raises the error.  With `wgrad.enabled`, the
    gradient of an fp32 table is added to its `.grad` in place, which touches the rows that occur and no others, wherever
    that changes nothing a user sees (`bagua_core_b200.ops.wgrad`)."""
    padding = -1
    if padding_idx is not None:
        rows = table.shape[0]
        if not -rows <= padding_idx < rows:
            raise ValueError(f"padding_idx {padding_idx} of a table of {rows} rows")
        padding = padding_idx % rows
    return _C.embedding(ids, table, scale, padding, dtype, _wgrad.active())


class ScaledEmbedding(nn.Embedding):
    """`nn.Embedding` times `scale`, through `embedding`; `dtype_out`: what it gives (under autocast by default autocast's type,
    else the table's).  Without the options that change rows while they are looked up or count them (`max_norm`,
    `scale_grad_by_freq`, `sparse`)."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx: Optional[int] = None,
                 dtype_out: Optional[torch.dtype] = None, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = scale
        self.dtype_out = dtype_out

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: Optional[int] = None, scale: float = 1.0,
                        dtype_out: Optional[torch.dtype] = None) -> "ScaledEmbedding":
        """One whose table is `embeddings`, as `nn.Embedding.from_pretrained` makes it."""
        if embeddings.dim() != 2:
            raise ValueError("a table has rows and columns")
        made = cls(*embeddings.shape, scale=scale, padding_idx=padding_idx, dtype_out=dtype_out, device="meta")
        made.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return made

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        dtype, dev = self.dtype_out, ids.device.type
        if dtype is None and torch.is_autocast_enabled(dev):
            dtype = torch.get_autocast_dtype(dev)
        return embedding(ids, self.weight, self.scale, self.padding_idx, dtype)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale}"
