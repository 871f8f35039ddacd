"""Embedding lookup with a scale and learned positions in one kernel, and the dense gradients of both tables.

The reference's language model adds two ``nn.Embedding`` modules (train.py:78-79,120-123).  The CUDA kernels sit behind
``sa2_embed_fwd`` / ``sa2_embed_bwd`` in ``include/sa2.h``; the autograd node is native (``csrc/sa2_torch.cpp``).
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)


def token_embedding(tokens: Tensor, weight: Tensor, pos_weight: Tensor | None = None, *, scale: float = 1.0, start: int = 0,
                    padding_idx: int | None = None) -> Tensor:
    """``scale * weight[tokens] + pos_weight[start : start + n]``, computed in fp32 and rounded once.

    ``tokens``: int64 or int32, ``(..., n)``; ``weight``: ``(vocab, dim)``, fp32 or bf16; ``pos_weight``: ``(positions, dim)`` of the same
    dtype, of which the last dimension of ``tokens`` takes rows ``start`` on.  A token outside ``[0, vocab)`` reads nothing: its row is
    NaN, and it has no gradient.  The gradients are dense; sums run over the sorted tokens in fp32 in one order, so that they are the
    same bits from run to run.  The row ``padding_idx`` of the table (negative: from its end, as in ``nn.Embedding``)
    gets no gradient."""
    padding = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None and weight.dim() == 2:
        if not -weight.shape[0] <= padding < weight.shape[0]:
            raise ValueError(f"padding_idx {padding} is outside of the table")
        padding %= weight.shape[0]
    out = _lib.ext().embed(tokens, weight, pos_weight, float(scale), int(start), padding)
    if out is not None:
        return out
    tensors = [t for t in (tokens, weight, pos_weight) if t is not None]
    assert all(t.is_cuda for t in tensors), "token_embedding needs CUDA tensors"
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32, not {tokens.dtype}")
    if weight.dtype not in _DTYPES or any(t.dtype != weight.dtype for t in tensors[1:]):
        raise ValueError("the tables must share one dtype, float32 or bfloat16")
    if any(t.dim() != 2 for t in tensors[1:]) or weight.numel() == 0 or any(t.shape[1] != weight.shape[1] for t in tensors[1:]):
        raise ValueError("expected tables of (rows, dim), with one dim and at least one row")
    if weight.shape[1] > 2 ** 30:
        raise ValueError("rows of a table may have up to 2^30 channels")
    if pos_weight is not None and not 0 <= start <= pos_weight.shape[0] - (tokens.shape[-1] if tokens.dim() else 1):
        raise ValueError("the positions do not fit the table of positions")
    raise RuntimeError("token_embedding takes plain tensors of one device, outside of tracing and transforms")
