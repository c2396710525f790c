"""Token embeddings shared with the output head (``genesis/model/embeddings.py:13-56``).

On CUDA the lookup, its scaling and its gradient are the kernels of
``llm_research_b200.ops.embedding``.  ``scale`` (an extension) multiplies the
looked-up rows, not the head that shares the table.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from llm_research_b200 import ops


class SharedEmbeddings(nn.Module):
    def __init__(self, vocab_size: int, d_model: int, dropout: float = 0.0, padding_idx: int | None = None,
                 scale: float = 1.0) -> None:
        super().__init__()
        self.d_model = d_model
        self.scale = scale
        self.embedding = nn.Embedding(vocab_size, d_model, padding_idx=padding_idx)
        self.dropout = nn.Dropout(dropout) if dropout > 0.0 else nn.Identity()

    @property
    def weight(self) -> torch.Tensor:
        return self.embedding.weight

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        w = self.embedding.weight
        if w.is_cuda and w.dtype in (torch.bfloat16, torch.float16, torch.float32):
            return self.dropout(ops.embedding(input_ids, w, self.scale, self.embedding.padding_idx))
        out = self.embedding(input_ids)
        return self.dropout(out if self.scale == 1.0 else out * self.scale)
