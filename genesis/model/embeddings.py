"""Token embeddings shared with the output head (``genesis/model/embeddings.py:13-56``).

On CUDA the lookup, its scaling and its gradient are the kernels of
``llm_research_b200.ops.embedding``.  ``scale`` (an extension) multiplies the
looked-up rows, not the head that shares the table.

The kernels stand in for the inner ``nn.Embedding`` only where that computes nothing
else than the lookup and nobody watches it: with hooks on it, another module or
``forward`` in its place, ``max_norm``, ``sparse`` or ``scale_grad_by_freq`` set, under
function transforms (vmap, ``torch.func``) and tracing, and for tensor subclasses, the
module itself is called.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from llm_research_b200 import ops

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _table(e: nn.Module, input_ids: torch.Tensor) -> torch.Tensor | None:
    """The weight where ``e(input_ids)`` is the plain lookup of plain CUDA tensors, unobserved."""
    if type(input_ids) is not torch.Tensor or type(e) is not nn.Embedding:
        return None
    d = e.__dict__
    if (d["_forward_hooks"] or d["_forward_pre_hooks"] or d["_backward_hooks"] or d["_backward_pre_hooks"]
            or "forward" in d or d["max_norm"] is not None or d["sparse"] or d["scale_grad_by_freq"]):
        return None
    w = e.weight
    if not w.is_cuda or w.dtype not in _DTYPES or type(w) not in (nn.Parameter, torch.Tensor):
        return None
    if (_has_any_global_hook() or torch.compiler.is_compiling() or torch.jit.is_tracing()
            or torch._C._len_torch_dispatch_stack() or torch._C._functorch.peek_interpreter_stack() is not None):
        return None
    return w


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
        if torch.jit.is_scripting():
            return self.dropout(self.embedding(input_ids) * self.scale)
        else:
            e = self.embedding
            w = _table(e, input_ids)
            if w is not None:
                return self.dropout(ops.embedding(input_ids, w, self.scale, e.padding_idx))
            out = e(input_ids)
            return self.dropout(out if self.scale == 1.0 else out * self.scale)
