"""Distillation from a teacher's largest logits: the loss of a position, and the gradient of the student's logits.

The reference trains on next tokens alone (train.py:129-135).  The CUDA kernels sit behind ``sa2_distill_fwd`` / ``sa2_distill_bwd`` /
``sa2_distill_both`` in ``include/sa2.h``; the autograd node is native (``csrc/sa2_torch.cpp``).
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)
_REDUCTIONS = {"sum": 0, "mean": 1, "none": 2}


def _refuse(logits, teacher_logits, teacher_index, temperature, reduction, reductions):
    assert all(t.is_cuda for t in (logits, teacher_logits, teacher_index)), "distillation needs CUDA tensors"
    if logits.dtype not in _DTYPES or teacher_logits.dtype not in _DTYPES or teacher_index.dtype not in (torch.int64, torch.int32):
        raise ValueError("logits must be float32 or bfloat16, the teacher's indices int64 or int32")
    if logits.dim() < 1 or teacher_logits.shape != teacher_index.shape or teacher_logits.shape[:-1] != logits.shape[:-1]:
        raise ValueError("expected logits of (..., vocab) and the teacher's logits and indices of (..., k)")
    if not 1 <= logits.shape[-1] <= 2 ** 30 or not 1 <= teacher_logits.shape[-1] <= 1024:
        raise ValueError("the vocabulary must have 1 to 2^30 entries, and the teacher 1 to 1024")
    raise RuntimeError("distillation takes plain tensors of one device, outside of tracing and transforms")


def _check(temperature, reduction, reductions):
    if not 5e-39 <= temperature <= 3e38:                 # fp32 in the kernels, and its inverse
        raise ValueError(f"temperature must be positive and finite, not {temperature}")
    if reduction not in reductions:
        raise ValueError(f"reduction must be one of {', '.join(reductions)}, not {reduction!r}")


def distillation_loss(logits: Tensor, teacher_logits: Tensor, teacher_index: Tensor, *, temperature: float = 1.0, reduction: str = "mean") -> Tensor:
    """``T^2 KL(p || q)`` of every row: ``q = softmax(logits / T)`` over the vocabulary, ``p = softmax(teacher_logits / T)`` over the
    teacher's k entries of the row, which stand at ``teacher_index``.

    ``logits``: ``(..., vocab)``, fp32 or bf16; ``teacher_logits``, ``teacher_index``: ``(..., k)``, k up to 1024.  Entries whose index lies
    outside ``[0, vocab)`` (say -1) are not there, whatever their logit; a row without entries, or whose entries are all -inf, has loss
    and gradient zero and does not count in the mean.  Entries of one token add up.  The result is fp32: the mean over the rows that
    count (0 if none does), their ``"sum"``, or with ``"none"`` one value for each row.  Gradients flow to ``logits``.

    A row's sum of exponentials is fp32: however near the student is to its teacher, the loss is good to about ``2^-21 T^2``, no better."""
    _check(temperature, reduction, _REDUCTIONS)
    loss = _lib.ext().distill(logits, teacher_logits, teacher_index, float(temperature), _REDUCTIONS[reduction])
    return loss if loss is not None else _refuse(logits, teacher_logits, teacher_index, temperature, reduction, _REDUCTIONS)


def distillation_loss_and_grad(logits: Tensor, teacher_logits: Tensor, teacher_index: Tensor, *, temperature: float = 1.0, reduction: str = "mean",
                               grad_scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """The loss of ``distillation_loss`` (``"mean"`` or ``"sum"``) and the gradient of ``logits`` times ``grad_scale`` from one call, for a step
    that goes backward at once: ``logits.backward(grad)``.  It reads the logits from memory once where autograd's two calls read them twice.
    ``grad_scale`` is what the loss would be multiplied with before its backward (a loss scale, one over accumulated steps)."""
    _check(temperature, reduction, ("mean", "sum"))
    if not abs(grad_scale) <= torch.finfo(torch.float32).max:           # fp32 in the kernels
        raise ValueError(f"grad_scale must be finite in fp32, not {grad_scale}")
    res = _lib.ext().distill_both(logits, teacher_logits, teacher_index, float(temperature), _REDUCTIONS[reduction], float(grad_scale))
    return res if res is not None else _refuse(logits, teacher_logits, teacher_index, temperature, reduction, _REDUCTIONS)
