"""Token embedding with scaling, and its gradient by sorted tokens.

``out[n] = scale * weight[ids[n]]`` and
``dW[v] = scale * sum of dout[n] over the n with ids[n] = v`` -- products and
sums in fp32, one rounding to the weight's dtype (bf16, fp16 or fp32).

CUDA (``csrc/kernels/embedding.cu``): the lookup is one kernel; the gradient
sorts the tokens (one cluster, stable) and adds the occurrences of a token in the
order of their positions: the same inputs give the same bits.  The lookup and its
gradient carry forward-mode tangents, and can be differentiated again.
``padding_idx`` only leaves its row out of the gradient (``F.embedding`` semantics).  An id outside ``[0, V)`` cannot be reported from
the device without a synchronisation: its output row is NaN and it has no
gradient (on the CPU it raises ``IndexError``).
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from llm_research_b200._ext import native

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``, shape ``(*ids.shape, d)``; ``ids`` int64 or int32 of any
    shape, ``weight`` ``(V, d)``.  See the module docstring."""
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight must be (V, d), got {tuple(weight.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    V, scale = weight.shape[0], float(scale)
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} outside the table of {V} rows")
        padding_idx %= V
    if not weight.is_cuda:
        out = F.embedding(ids, weight, padding_idx)
        if scale == 1.0:
            return out
        return out * scale if out.dtype in (torch.float32, torch.float64) else (out.float() * scale).to(out.dtype)
    if weight.dtype not in _DTYPES:
        raise TypeError(f"embedding: weight must be bf16, fp16 or fp32 on CUDA, got {weight.dtype}")
    return native().embedding(ids, weight, scale, -1 if padding_idx is None else padding_idx)
