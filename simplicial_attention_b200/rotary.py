"""RMSNorm of every query and key head and the rotation by position behind it, in one kernel.

The reference's standard layers have neither (two_simplicial_transformer.py:25-65); its sliding-window module has the norms alone
(simplicial_mha.py:69-73,124-127).  The CUDA kernels sit behind ``sa2_rotary_fwd`` / ``sa2_rotary_bwd`` in ``include/sa2.h``; the
autograd node is native (``csrc/sa2_torch.cpp``).
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)


def rotary_frequencies(rotated: int, theta: float = 10000.0, device=None, *, inv_freq: Tensor | None = None) -> Tensor:
    """What ``qk_norm_rotary`` turns by: one int64 for each of the ``rotated // 2`` pairs of channels, in 2^-64 turns per position.  Pair
    ``i`` turns by ``theta ** (-2 i / rotated)`` radians a position, or by ``inv_freq[i]`` (any other schedule, fp64)."""
    if inv_freq is None:
        if rotated <= 0 or rotated % 2:
            raise ValueError(f"rotated must be even and positive, not {rotated}")
        inv = [float(theta) ** (-2.0 * i / rotated) for i in range(rotated // 2)]
    else:
        if 2 * inv_freq.numel() != rotated:
            raise ValueError(f"expected {rotated // 2} frequencies, not {inv_freq.numel()}")
        inv = inv_freq.double().flatten().tolist()
    if not all(math.isfinite(f) for f in inv):
        raise ValueError("frequencies must be finite")
    turns = [round(f / (2 * math.pi) * 2.0 ** 64) for f in inv]
    return torch.tensor([(t + 2 ** 63) % 2 ** 64 - 2 ** 63 for t in turns], dtype=torch.int64, device=device)


def qk_norm_rotary(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, freqs: Tensor, *, start: int = 0, positions: Tensor | None = None,
                   eps: float | None = None, interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """``(q, k)`` normalised per head - ``x * rsqrt(mean(x^2) + eps) * weight``, as ``torch.nn.RMSNorm(d)`` - and turned by position.

    ``q``: ``(b, n, hq, d)``, ``k``: ``(b, n, hk, d)``, fp32 or bf16, with any strides in front of a contiguous last dimension (views into a
    packed projection are read in place); d is 32, 64, 128 or 256.  ``q_weight``, ``k_weight``: ``(d,)``.  ``freqs``: from
    ``rotary_frequencies(rotated)``, rotated a multiple of 16 up to d; channels from ``rotated`` on are only normalised.  Pairs are
    channels ``(i, i + rotated / 2)``, or ``(2 i, 2 i + 1)`` if ``interleaved``.  Row ``i`` is at position ``start + i``, or at
    ``positions`` - int64, ``(n,)`` or ``(b, n)``, any value: the angle is exact modulo a turn.  ``eps`` defaults to the dtype's machine epsilon.
    Results are ``(b, n, heads, d)``, contiguous, in the dtype of ``q`` and ``k``; everything in between is fp32."""
    eps = float(eps) if eps is not None else torch.finfo(q.dtype).eps if q.dtype in _DTYPES else 0.0
    res = _lib.ext().qk_norm_rotary(q, k, q_weight, k_weight, freqs, positions, int(start), eps, bool(interleaved))
    if res is not None:
        return res
    tensors = [t for t in (q, k, q_weight, k_weight, freqs, positions) if t is not None]
    assert all(t.is_cuda for t in tensors), "qk_norm_rotary needs CUDA tensors"
    if q.dtype not in _DTYPES or k.dtype != q.dtype or q_weight.dtype not in _DTYPES or k_weight.dtype != q_weight.dtype:
        raise ValueError("q and k must share one dtype and so must their weights: float32 or bfloat16")
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.shape[2] == 0 or k.shape[2] == 0:
        raise ValueError("expected (batch, seq, heads, dim_head) queries and keys of the same rows")
    d = q.shape[3]
    if d not in (32, 64, 128, 256):
        raise ValueError(f"dim_head {d} is not supported (32, 64, 128 or 256)")
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        raise ValueError("each weight must have dim_head entries")
    if freqs.dtype != torch.int64 or freqs.dim() != 1 or freqs.numel() == 0 or freqs.numel() % 8 or 2 * freqs.numel() > d:
        raise ValueError("freqs must come from rotary_frequencies(rotated), rotated a multiple of 16 up to dim_head")
    if positions is not None and (positions.dtype != torch.int64 or positions.dim() not in (1, 2) or positions.shape[-1] != q.shape[1]
                                  or (positions.dim() == 2 and positions.shape[0] not in (1, q.shape[0]))):
        raise ValueError("positions must be int64 of (seq,) or (batch, seq)")
    raise RuntimeError("qk_norm_rotary takes plain tensors of one device (up to 2^30 rows, 4096 heads), outside of tracing and transforms")


def _turned(n, freqs, start, interleaved=False):
    """The rotation of rows at positions ``start`` on, in torch's operators: a function of fp32 heads ``(b, n, heads, d)``."""
    steps = torch.arange(start, start + n, device=freqs.device)[:, None, None] * freqs      # modulo a turn: int64 wraps
    angle = steps.double() * (math.pi * 2.0 ** -63)
    cos, sin = angle.cos().float(), angle.sin().float()
    rotated = 2 * freqs.numel()

    def turn(y):
        a, b = (y[..., 0:rotated:2], y[..., 1:rotated:2]) if interleaved else y[..., :rotated].chunk(2, -1)
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
        return torch.cat((turned, y[..., rotated:]), dim=-1)

    return turn


def _plain(q, k, q_weight, k_weight, freqs, start, eps, interleaved=False):
    """The same in torch's operators: CPU tensors, other head dims, and what torch records or transforms."""
    turn = _turned(q.shape[1], freqs, start, interleaved)

    def one(x, weight):
        y = x.float()
        return turn(y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)

    return one(q, q_weight), one(k, k_weight)
