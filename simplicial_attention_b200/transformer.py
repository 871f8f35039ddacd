"""Decoder stack and language-model wrapper around the sliding-window
2-simplicial attention module: the harness for the training-step configuration
(8 layers, dim 512, every 2nd layer simplicial, byte vocabulary).

Restates, in plain PyTorch, ``TwoSimplicialTransformer`` / ``Attention`` /
``FeedForward`` (simplicial_attention/two_simplicial_transformer.py:25-141) and
the ``TwoSimplicialLM`` wrapper of the reference's example script
(train.py:64-135; the script itself runs its training loop at import and needs
a dataset blob that is not shipped).  Parameter names match the reference, so
its checkpoints load.  The standard layers use torch's scaled-dot-product attention, as in the
reference; the RMSNorm modules are ``headnorm.RMSNorm`` (same parameter, fused CUDA kernel).  On CUDA
the embeddings are one kernel (``embedding.py``).  Beyond the reference: normalised and rotated queries and
keys in the standard layers, a scale on the embeddings, distillation from a teacher's largest logits, and
sampling with top-p and min-p.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch import nn
from torch.nn import Module, ModuleList
from torch.nn.modules.module import _has_any_global_hook

from . import _lib
from .attention import divisible_by
from .distill import distillation_loss, distillation_loss_and_grad
from .headnorm import RMSNorm
from .mha import SlidingWindowTwoSimplicialMHA, _child
from .rotary import _plain as plain_qk_norm_rotary
from .rotary import _turned as turned
from .rotary import rotary_frequencies
from .sampling import sample_tokens


def _hooked(m):
    """Whether a call of ``m`` runs more than its class's ``forward``."""
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks or "forward" in m.__dict__)


class Attention(Module):
    """Pre-norm causal grouped-query attention (two_simplicial_transformer.py:25-65).  With ``qk_norm_rotary`` (not in the reference)
    queries and keys are normalised per head and turned by position, in one kernel on CUDA."""

    qk_norm_rotary = False      # (of modules pickled without the option)

    def __init__(self, dim, dim_head=64, heads=8, key_value_heads=8, qk_norm_rotary=False, rotary_theta=10000.0):
        super().__init__()
        assert divisible_by(heads, key_value_heads)
        self.heads, self.key_value_heads, self.dim_head = heads, key_value_heads, dim_head
        self.prenorm = RMSNorm(dim)
        self.to_q = nn.Linear(dim, heads * dim_head, bias=False)
        self.to_kv = nn.Linear(dim, key_value_heads * dim_head * 2, bias=False)
        self.to_out = nn.Linear(heads * dim_head, dim, bias=False)
        self.qk_norm_rotary = qk_norm_rotary
        if qk_norm_rotary:
            self.q_norm, self.k_norm = RMSNorm(dim_head), RMSNorm(dim_head)
            self.register_buffer("freqs", rotary_frequencies(dim_head, rotary_theta), persistent=False)

    def _norm_rotate(self, q, k, start):
        """One native call, or its plain form; the modules themselves where one is not a plain ``RMSNorm`` of a head (another type, a hook) or
        they are not alike."""
        norms = _child(self, "q_norm"), _child(self, "k_norm")
        if _has_any_global_hook() or any(type(m) is not RMSNorm or m.dim != self.dim_head or _hooked(m) for m in norms) or norms[0].eps != norms[1].eps:
            q, k = self.q_norm(q), self.k_norm(k)
            turn = turned(q.shape[1], self.freqs, start)
            return turn(q.float()).to(q.dtype), turn(k.float()).to(k.dtype)
        eps = norms[0].eps if norms[0].eps is not None else torch.finfo(torch.float32 if torch.is_autocast_enabled() else q.dtype).eps
        args = (q, k, _child(norms[0], "weight"), _child(norms[1], "weight"), self.freqs)
        res = _lib.ext().qk_norm_rotary(*args, None, start, eps, False) if q.is_cuda else None
        return res if res is not None else plain_qk_norm_rotary(*args, start, eps)

    def forward(self, x, cache=None, return_cache=False):
        """``cache`` = (keys, values) of every earlier position; with a cache ``x`` is one new position."""
        b, n, _ = x.shape
        x = self.prenorm(x)
        q = self.to_q(x).view(b, n, self.heads, self.dim_head)
        # the fused projection is laid out (kv, h, d), as in the reference's rearrange
        kv = self.to_kv(x).view(b, n, 2, self.key_value_heads, self.dim_head)
        k = kv[:, :, 0]
        if self.qk_norm_rotary:
            q, k = self._norm_rotate(q, k, 0 if cache is None else cache[0].shape[2])
        q, k, v = q.transpose(1, 2), k.transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        if cache is not None:
            assert n == 1, "with a cache, feed one new position at a time"
            k, v = torch.cat((cache[0], k), dim=2), torch.cat((cache[1], v), dim=2)
        out = F.scaled_dot_product_attention(q, k, v, is_causal=cache is None, enable_gqa=self.heads != self.key_value_heads)
        out = self.to_out(out.transpose(1, 2).reshape(b, n, -1))
        return (out, (k.detach(), v.detach())) if return_cache else out


def FeedForward(dim, expansion=4.0):
    inner = int(dim * expansion)
    return nn.Sequential(RMSNorm(dim), nn.Linear(dim, inner), nn.GELU(), nn.Linear(inner, dim))


class TwoSimplicialTransformer(Module):
    def __init__(self, dim, *, depth, heads=8, key_value_heads=4, dim_head=64, ff_expansion=4.0,
                 two_simplicial_attn_every=4, attn_kwargs: dict = dict(),
                 two_simplicial_attn_kwargs: dict = dict(w1=512, w2=32, qk_rmsnorm=True), final_norm=True):
        super().__init__()
        layers = []
        for index in range(depth):
            if divisible_by(index + 1, two_simplicial_attn_every):
                attn = SlidingWindowTwoSimplicialMHA(dim=dim, heads=heads, key_value_heads=key_value_heads,
                                                     dim_head=dim_head, prenorm=True, **two_simplicial_attn_kwargs)
            else:
                attn = Attention(dim=dim, heads=heads, key_value_heads=key_value_heads, dim_head=dim_head, **attn_kwargs)
            layers.append(ModuleList([attn, FeedForward(dim=dim, expansion=ff_expansion)]))
        self.layers = ModuleList(layers)
        self.norm = RMSNorm(dim) if final_norm else nn.Identity()

    def forward(self, x, cache=None, return_cache=False):
        """``cache``: one entry per layer, as returned by an earlier call with ``return_cache=True``."""
        if cache is None and not return_cache:
            for attn, ff in self.layers:
                x = attn(x) + x
                x = ff(x) + x
            return self.norm(x)
        new_cache = []
        for index, (attn, ff) in enumerate(self.layers):
            a, c = attn(x, cache=None if cache is None else cache[index], return_cache=True)
            new_cache.append(c)
            x = a + x
            x = ff(x) + x
        return self.norm(x), new_cache


class TwoSimplicialLM(Module):
    """Token + learned absolute position embedding, the decoder stack, a linear head
    (train.py:64-135).  ``forward(x, return_loss=True)`` takes ``(b, n + 1)`` token ids and
    returns the next-token cross entropy; with a teacher's largest logits ``(b, n, k)`` and where they stand
    it returns ``distillation_loss`` against those instead (CUDA, fp32 or bf16 logits).  On CUDA a token outside of the table has NaN for an
    embedding, and ``sample_tokens`` answers -1 for logits of NaN; on the CPU it is torch's ``IndexError``."""

    embed_scale = 1.0           # (of modules pickled without the option)

    def __init__(self, *, num_tokens, dim, depth, max_seq_len=1024, dim_head=64, heads=8,
                 two_simplicial_attn_every=4, transformer_kwargs=dict(), embed_scale=1.0):
        super().__init__()
        self.embed_scale = embed_scale
        self.token_emb = nn.Embedding(num_tokens, dim)
        self.pos_emb = nn.Embedding(max_seq_len, dim)
        self.transformer = TwoSimplicialTransformer(dim=dim, depth=depth, dim_head=dim_head, heads=heads,
                                                    two_simplicial_attn_every=two_simplicial_attn_every,
                                                    **transformer_kwargs)
        self.to_logits = nn.Linear(dim, num_tokens, bias=False)

    def _embed(self, x, start):
        """Token and position embeddings of rows ``start`` on: one native call, or the two modules where one of them is not a plain
        ``nn.Embedding`` (another type, an option, a hook) or the call declines."""
        te, pe = _child(self, "token_emb"), _child(self, "pos_emb")
        if type(pe) is nn.Embedding and not _hooked(pe) and start + x.shape[-1] > pe.num_embeddings:
            raise IndexError(f"{start + x.shape[-1]} rows are more than the table's {pe.num_embeddings} positions")
        plain = x.is_cuda and not _has_any_global_hook() and all(
            type(m) is nn.Embedding and m.max_norm is None and not m.scale_grad_by_freq and not m.sparse and m.padding_idx is None and not _hooked(m)
            for m in (te, pe))
        if plain:
            res = _lib.ext().embed(x, _child(te, "weight"), _child(pe, "weight"), float(self.embed_scale), start, -1)
            if res is not None:
                return res
        tokens = self.token_emb(x)
        if self.embed_scale != 1.0:
            tokens = tokens * self.embed_scale
        return tokens + self.pos_emb(torch.arange(start, start + x.shape[-1], device=x.device))

    def forward(self, x, return_loss=False, cache=None, return_cache=False, teacher_logits=None, teacher_index=None, temperature=1.0):
        if (teacher_logits is None) != (teacher_index is None):
            raise ValueError("a teacher has logits and an index")
        if teacher_logits is not None and (not return_loss or return_cache):
            raise ValueError("a teacher is for the loss: return_loss=True, without a cache")
        if return_loss:
            x, target = x[:, :-1], x[:, 1:]
        n = x.shape[-1]
        start = 0 if cache is None else cache["length"]
        tokens = self._embed(x, start)
        if cache is None and not return_cache:
            logits = self.to_logits(self.transformer(tokens))
        else:
            embed, layers = self.transformer(tokens, cache=None if cache is None else cache["layers"], return_cache=True)
            logits = self.to_logits(embed)
            return logits, {"length": start + n, "layers": layers}
        if not return_loss:
            return logits
        if teacher_logits is not None:
            return distillation_loss(logits, teacher_logits, teacher_index, temperature=temperature)
        return F.cross_entropy(logits.transpose(1, 2), target)

    @torch.no_grad()
    def sample(self, prompt: torch.Tensor, seq_len: int, temperature=1.0, filter_thres=0.9, use_cache=True, *, top_k=None, top_p=None,
               min_p=None, generator=None):
        """Same contract as the reference's ``sample`` (train.py:92-111): top-k filtered Gumbel sampling
        until ``seq_len`` tokens, returning only the generated part.  With ``use_cache`` the prompt is run
        once and every further token costs one position: the standard layers keep their keys and values,
        the simplicial layers only their ``w1 - 1`` / ``w2 - 1`` row windows.  With any of ``top_k``, ``top_p`` and ``min_p`` the tokens
        come from ``sample_tokens`` (``filter_thres`` is then not used; it needs CUDA and fp32 or bf16 logits).  Random numbers come from
        ``generator``, or torch's own."""
        filtered = top_k is not None or top_p is not None or min_p is not None
        out = prompt.clone()
        steps = max(0, seq_len - prompt.shape[-1])
        cache = None
        for step in range(steps):
            if not use_cache:
                logits = self.forward(out)
            elif cache is None:
                logits, cache = self.forward(out, return_cache=True)
            else:
                logits, cache = self.forward(out[:, -1:], cache=cache, return_cache=True)
            if filtered:
                uniform = torch.rand(out.shape[0], device=out.device, generator=generator)
                nxt = sample_tokens(logits[:, -1], uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
                out = torch.cat((out, nxt[:, None]), dim=-1)
                continue
            logits = logits[:, -1].float()
            k = max(1, math.ceil((1 - filter_thres) * logits.shape[-1]))
            val, ind = torch.topk(logits, k)
            kept = torch.full_like(logits, float("-inf")).scatter_(-1, ind, val)
            uniform = torch.rand(kept.shape, device=kept.device, generator=generator)
            noise = -torch.log((-torch.log(uniform.clamp_min(1e-20))).clamp_min(1e-20))
            nxt = (kept / max(temperature, 1e-10) + noise).argmax(dim=-1, keepdim=True)
            out = torch.cat((out, nxt), dim=-1)
        return out[..., prompt.shape[-1]:]


def training_step(model: Module, optimizer: torch.optim.Optimizer, tokens: torch.Tensor, max_grad_norm=0.5, *, teacher_logits=None, teacher_index=None,
                  temperature=1.0) -> torch.Tensor:
    """One step of the reference's loop (train.py:179-194, without gradient accumulation):
    loss, backward, clip to 0.5, Adam step.  Returns the loss tensor (no host sync).  With a teacher's largest logits ``(b, n, k)`` for the
    ``n`` positions before the last token, and where they stand, the loss is ``distillation_loss`` against those."""
    if (teacher_logits is None) != (teacher_index is None):
        raise ValueError("a teacher has logits and an index")
    if teacher_logits is None:
        loss = model(tokens, return_loss=True)
        loss.backward()
    else:
        logits = model(tokens[:, :-1])
        loss, grad = distillation_loss_and_grad(logits, teacher_logits, teacher_index, temperature=temperature)
        logits.backward(grad)
    torch.nn.utils.clip_grad_norm_(model.parameters(), max_grad_norm)
    optimizer.step()
    optimizer.zero_grad(set_to_none=True)
    return loss
