"""A token for each row of logits: temperature, top-k, top-p and min-p in one kernel, from given random numbers.

The reference's ``sample`` filters by top-k alone, with a chain of torch calls a token (train.py:39-60,104-109).  The CUDA kernel sits
behind ``sa2_sample`` in ``include/sa2.h``.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)


def _setting(value, name, rows, logits, dtype):
    """A tensor of a value for each row as the kernel reads it."""
    if not isinstance(value, Tensor):
        return value
    if value.is_floating_point() != dtype.is_floating_point or value.dtype == torch.bool or value.is_complex():
        raise ValueError(f"{name}: expected {'floating-point' if dtype.is_floating_point else 'whole'} numbers, not {value.dtype}")
    if value.shape != rows:
        raise ValueError(f"{name}: expected a value for each row, shape {tuple(rows)}, not {tuple(value.shape)}")
    if value.device != logits.device:
        raise ValueError(f"{name} must be on the device of the logits")
    return value.to(dtype).contiguous()


def sample_tokens(logits: Tensor, uniform: Tensor, *, temperature=1.0, top_k=None, top_p=None, min_p=None, return_logprobs: bool = False):
    """One token for each row of ``logits`` ``(..., vocab)``, fp32 or bf16, drawn with the row's number of ``uniform`` ``(...)``, fp32 or fp64
    in ``[0, 1)``: int64 ``(...)``; with ``return_logprobs`` also the fp32 logarithm of the probability that the token had.

    Tokens rank by logit, equal ones by index.  ``softmax(logits / temperature)`` is cut to the ``top_k`` first tokens; then to those
    before which less than ``top_p`` of the remaining mass has come; then to those at least ``min_p`` times as probable as the best.  The
    best token always stays.  What is left is drawn from by its running mass in the order of the indices: the first token at
    which it exceeds ``uniform`` times the whole.  A temperature of 0 takes the best token.  Each setting is a number or a tensor of one
    for each row; ``None`` is off, and so are ``top_k <= 0``, ``top_p >= 1`` and ``min_p <= 0``.

    The result is a function of the arguments alone: the same for a row whatever the rows beside it.  A row that holds a NaN or +inf,
    or nothing above -inf, has no distribution: token -1, log-probability NaN."""
    t, k, p, m = (None if isinstance(v, Tensor) else off if v is None else v for v, off in ((temperature, 1.0), (top_k, 0), (top_p, 1.0), (min_p, 0.0)))
    for name, value in (("temperature", t), ("top_p", p), ("min_p", m)):
        if value is not None and not 0 <= value < math.inf:
            raise ValueError(f"{name} must be finite and not negative, not {value}")
    numbers = (1.0 if t is None else float(t), 0 if k is None else int(k), 1.0 if p is None else float(p), 0.0 if m is None else float(m))

    def call(t, k, p, m):
        return _lib.ext().sample(logits, uniform, t, numbers[0], k, numbers[1], p, numbers[2], m, numbers[3], bool(return_logprobs))

    res = call(*(v if isinstance(v, Tensor) else None for v in (temperature, top_k, top_p, min_p)))
    if res is None:
        # tensors of other types, or what cannot be taken
        assert logits.is_cuda and uniform.is_cuda, "sample_tokens needs CUDA tensors"
        if logits.dtype not in _DTYPES or uniform.dtype not in (torch.float32, torch.float64):
            raise ValueError("logits must be float32 or bfloat16, uniform float32 or float64")
        rows = logits.shape[:-1]
        if logits.dim() < 1 or not 1 <= logits.shape[-1] <= 2 ** 30 or uniform.shape != rows:
            raise ValueError("expected logits of (..., vocab), vocab up to 2^30, and a uniform number for each row")
        res = call(*(v if isinstance(v, Tensor) else None for v in (
            _setting(temperature, "temperature", rows, logits, torch.float32), _setting(top_k, "top_k", rows, logits, torch.int64),
            _setting(top_p, "top_p", rows, logits, torch.float32), _setting(min_p, "min_p", rows, logits, torch.float32))))
        if res is None:
            raise RuntimeError("sample_tokens takes plain tensors of one device, outside of tracing and transforms")
    return res if return_logprobs else res[0]
