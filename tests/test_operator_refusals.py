"""What the operators around the attention layers refuse, with the exceptions they name.  No kernel is launched: these run without a GPU."""
import ctypes as C
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import simplicial_attention_b200 as sa
from simplicial_attention_b200 import _lib, rotary


def _cuda(*shape, dtype=torch.float32):
    """A tensor that says it is on a GPU; its values are nowhere."""
    with FakeTensorMode():
        return torch.empty(shape, dtype=dtype, device="cuda")


def test_cpu_tensors():
    w, ids, u = torch.randn(4, 8), torch.zeros(2, 3, dtype=torch.long), torch.rand(2)
    with pytest.raises(AssertionError, match="CUDA"):
        sa.token_embedding(ids, w)
    with pytest.raises(AssertionError, match="CUDA"):
        sa.qk_norm_rotary(torch.randn(1, 2, 1, 64), torch.randn(1, 2, 1, 64), torch.ones(64), torch.ones(64), sa.rotary_frequencies(64))
    with pytest.raises(AssertionError, match="CUDA"):
        sa.distillation_loss(torch.randn(2, 9), torch.randn(2, 3), ids[:, :3])
    with pytest.raises(AssertionError, match="CUDA"):
        sa.distillation_loss_and_grad(torch.randn(2, 9), torch.randn(2, 3), ids[:, :3])
    with pytest.raises(AssertionError, match="CUDA"):
        sa.sample_tokens(torch.randn(2, 9), u)


def test_embedding():
    ids, w, p = _cuda(2, 3, dtype=torch.long), _cuda(9, 8), _cuda(5, 8)
    for args, kw, what in [((ids.float(), w), {}, "int64"), ((ids, w.half()), {}, "dtype"), ((ids, w, p.bfloat16()), {}, "dtype"), ((ids, w, _cuda(5, 7)), {}, "dim"),
                           ((ids, _cuda(8)), {}, "dim"), ((ids, _cuda(0, 8)), {}, "dim"), ((ids, w, p), dict(start=3), "positions"), ((ids, w, p), dict(start=-1), "positions")]:
        with pytest.raises(ValueError, match=what):
            sa.token_embedding(*args, **kw)
    for padding in (9, -10):
        with pytest.raises(ValueError, match="padding_idx"):
            sa.token_embedding(ids, w, padding_idx=padding)
    with pytest.raises(RuntimeError, match="plain tensors"):
        sa.token_embedding(ids, w, p)                    # no values to read


def test_rotary():
    q, k, g, f = _cuda(2, 5, 4, 64), _cuda(2, 5, 2, 64), _cuda(64), _cuda(32, dtype=torch.long)
    bad = [((q.half(), k.half(), g, g, f), {}, "float32"), ((q, k.bfloat16(), g, g, f), {}, "dtype"), ((q, k, g, g.bfloat16(), f), {}, "dtype"),
           ((q, _cuda(2, 4, 2, 64), g, g, f), {}, "rows"), ((q, _cuda(2, 5, 2, 32), g, g, f), {}, "rows"), ((q[0], k[0], g, g, f), {}, "batch"),
           ((_cuda(2, 5, 4, 48), _cuda(2, 5, 4, 48), _cuda(48), _cuda(48), f), {}, "dim_head"), ((q, k, g, _cuda(32), f), {}, "weight"),
           ((q, k, g, g, _cuda(40, dtype=torch.long)), {}, "freqs"), ((q, k, g, g, _cuda(12, dtype=torch.long)), {}, "freqs"), ((q, k, g, g, _cuda(32)), {}, "freqs"),
           ((q, k, g, g, f), dict(positions=_cuda(5)), "positions"), ((q, k, g, g, f), dict(positions=_cuda(4, dtype=torch.long)), "positions"),
           ((q, k, g, g, f), dict(positions=_cuda(3, 5, dtype=torch.long)), "positions")]
    for args, kw, what in bad:
        with pytest.raises(ValueError, match=what):
            sa.qk_norm_rotary(*args, **kw)
    with pytest.raises(RuntimeError, match="plain tensors"):
        sa.qk_norm_rotary(q, k, g, g, f)
    with pytest.raises(ValueError):
        sa.rotary_frequencies(15)
    with pytest.raises(ValueError):
        sa.rotary_frequencies(16, inv_freq=torch.ones(4))
    with pytest.raises(ValueError):
        sa.rotary_frequencies(16, inv_freq=torch.full((8,), math.inf))


@pytest.mark.parametrize("call", [sa.distillation_loss, sa.distillation_loss_and_grad])
def test_distillation(call):
    z, t, i = _cuda(4, 50), _cuda(4, 3), _cuda(4, 3, dtype=torch.long)
    for temperature in (0.0, -1.0, 1e-40, 1e39, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            call(z, t, i, temperature=temperature)
    with pytest.raises(ValueError, match="reduction"):
        call(z, t, i, reduction="median")
    for args, what in [((z.half(), t, i), "float32"), ((z, t.half(), i), "float32"), ((z, t, i.float()), "int64"), ((z, t, i[:, :2]), "k"), ((z[:3], t, i), "vocab"),
                       ((z, _cuda(4, 1025), _cuda(4, 1025, dtype=torch.long)), "1024"), ((z, _cuda(4, 0), _cuda(4, 0, dtype=torch.long)), "1024"), ((z[:, :0], t, i), "vocab")]:
        with pytest.raises(ValueError, match=what):
            call(*args)
    with pytest.raises(RuntimeError, match="plain tensors"):
        call(z, t, i)
    if call is sa.distillation_loss_and_grad:
        with pytest.raises(ValueError, match="reduction"):
            call(z, t, i, reduction="none")
        with pytest.raises(ValueError, match="grad_scale"):
            call(z, t, i, grad_scale=math.nan)


def test_sampling():
    z, u = _cuda(4, 50), _cuda(4)
    for kw, what in [(dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(top_p=-0.1), "top_p"), (dict(min_p=math.inf), "min_p"),
                     (dict(top_k=_cuda(4)), "top_k"), (dict(top_p=_cuda(4, dtype=torch.long)), "top_p"), (dict(top_p=_cuda(3)), "top_p"), (dict(min_p=torch.rand(4)), "min_p"),
                     (dict(top_k=_cuda(4, dtype=torch.bool)), "top_k")]:
        with pytest.raises(ValueError, match=what):
            sa.sample_tokens(z, u, **kw)
    for args, what in [((z.half(), u), "float32"), ((z, u.bfloat16()), "float32"), ((z, u[:3]), "row"), ((z[:, :0], u), "vocab")]:
        with pytest.raises(ValueError, match=what):
            sa.sample_tokens(*args)
    with pytest.raises(RuntimeError, match="plain tensors"):
        sa.sample_tokens(z, u)


class EmbedArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("tokens", "weight", "positions", "out", "dout", "dweight", "dpositions", "workspace")] + [("workspace_bytes", C.c_size_t)] + \
        [(n, C.c_int64) for n in ("rows", "vocab", "start", "position_rows", "padding")] + [(n, C.c_int32) for n in ("n", "dim", "dtype", "tokens64")] + \
        [("scale", C.c_float), ("stream", C.c_void_p)]


class SampleArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "uniform", "temperature", "top_p", "min_p", "top_k", "token", "logprob")] + \
        [(n, C.c_int64) for n in ("rows", "logits_stride", "top_k_all")] + [(n, C.c_double) for n in ("temperature_all", "top_p_all", "min_p_all")] + \
        [(n, C.c_int32) for n in ("vocab", "dtype", "uniform64")] + [("stream", C.c_void_p)]


class DistillArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "teacher", "index", "row_loss", "total", "gout", "dlogits", "workspace")] + [("workspace_bytes", C.c_size_t)] + \
        [(n, C.c_int64) for n in ("rows", "logits_stride", "teacher_stride", "index_stride", "dlogits_stride")] + \
        [(n, C.c_int32) for n in ("vocab", "k", "dtype", "teacher_dtype", "index64", "reduction", "gout_rows")] + \
        [(n, C.c_float) for n in ("temperature", "grad_scale")] + [("stream", C.c_void_p)]


class RotarySide(C.Structure):
    _fields_ = [("x", C.c_void_p), ("dy", C.c_void_p), ("sx", _lib.Strides), ("sdy", _lib.Strides), ("y", C.c_void_p), ("gain", C.c_void_p), ("dgain", C.c_void_p),
                ("heads", C.c_int32)]


class RotaryArgs(C.Structure):
    _fields_ = [("q", RotarySide), ("k", RotarySide), ("freqs", C.c_void_p), ("positions", C.c_void_p)] + [(n, C.c_int64) for n in ("pos_batch", "pos_seq", "start")] + \
        [("partial", C.c_void_p), ("partial_bytes", C.c_size_t)] + [(n, C.c_int32) for n in ("b", "n", "d", "pairs", "interleaved", "dtype", "gain_dtype")] + \
        [("eps", C.c_float), ("stream", C.c_void_p)]


A = 4096            # an address that is never dereferenced: checks come before any launch


def test_c_calls_of_the_embedding():
    lib = _lib.lib()
    good = dict(tokens=A, weight=A, out=A, dout=A, dweight=A, workspace=A, workspace_bytes=1 << 20, rows=12, vocab=9, n=4, dim=8, padding=-1, scale=1.0)

    def both(fwd, bwd, **kw):
        a = EmbedArgs(**{**good, **kw})
        assert fwd is None or lib.sa2_embed_fwd(C.byref(a)) == fwd
        assert bwd is None or lib.sa2_embed_bwd(C.byref(a)) == bwd

    for kw in (dict(tokens=0), dict(rows=0), dict(vocab=0), dict(n=5), dict(n=0), dict(dim=0), dict(start=-1), dict(positions=A, dpositions=A, position_rows=3)):
        both(1, 1, **kw)
    both(2, 2, dtype=7)
    both(2, 2, rows=1 << 32)
    both(1, None, weight=0)
    both(1, None, out=0)
    both(None, 1, dout=0)
    both(None, 1, dweight=0)
    both(None, 1, dweight=A + 8)
    both(None, 3, workspace=0)
    both(None, 3, workspace=A + 128)
    both(None, 3, workspace_bytes=64)


def test_c_calls_of_sampling_and_distillation():
    lib = _lib.lib()
    for kw, status in [(dict(logits=0), 1), (dict(uniform=0), 1), (dict(token=0), 1), (dict(rows=0), 1), (dict(vocab=-1), 1), (dict(vocab=(1 << 30) + 1), 2), (dict(dtype=3), 2), (dict(logits=A + 2), 1)]:
        assert lib.sa2_sample(C.byref(SampleArgs(**{**dict(logits=A, uniform=A, token=A, rows=2, vocab=5), **kw}))) == status
    assert lib.sa2_sample(None) == 1
    good = dict(logits=A, teacher=A, index=A, row_loss=A, total=A, dlogits=A, workspace=A, workspace_bytes=1 << 20, rows=3, vocab=9, k=2, temperature=1.0)
    for kw, status in [(dict(logits=0), 1), (dict(rows=0), 1), (dict(workspace=0), 3), (dict(workspace=A + 16), 3), (dict(workspace_bytes=300), 3), (dict(vocab=0), 1), (dict(k=0), 1),
                       (dict(k=1025), 2), (dict(vocab=(1 << 30) + 1), 2), (dict(dtype=5), 2), (dict(teacher_dtype=5), 2), (dict(reduction=4), 2), (dict(temperature=0.0), 1), (dict(temperature=1e-40), 1), (dict(temperature=math.inf), 1),
                       (dict(temperature=math.nan), 1), (dict(logits=A + 2), 1)]:
        a = C.byref(DistillArgs(**{**good, **kw}))
        assert lib.sa2_distill_fwd(a) == status and lib.sa2_distill_bwd(a) == status and lib.sa2_distill_both(a) == status
    for kw in (dict(teacher=0), dict(index=0), dict(row_loss=0, total=0)):
        a = C.byref(DistillArgs(**{**good, **kw}))
        assert lib.sa2_distill_fwd(a) == 1 and lib.sa2_distill_both(a) == 1
    assert lib.sa2_distill_both(C.byref(DistillArgs(**{**good, "total": 0}))) == 1
    assert lib.sa2_distill_bwd(C.byref(DistillArgs(**{**good, "dlogits": 0}))) == 1
    assert lib.sa2_distill_both(C.byref(DistillArgs(**{**good, "gout": A}))) == 1
    assert lib.sa2_distill_fwd(None) == 1 and lib.sa2_distill_bwd(None) == 1 and lib.sa2_distill_both(None) == 1


def test_c_calls_of_the_rotation():
    lib = _lib.lib()
    lib.sa2_rotary_partial_bytes.restype = C.c_size_t
    side = dict(x=A, y=A, dy=A, gain=A, dgain=A, heads=2, sx=_lib.Strides(640, 128, 64), sdy=_lib.Strides(640, 128, 64))
    good = dict(freqs=A, b=2, n=5, d=64, pairs=32, partial=A, partial_bytes=1 << 20)

    def run(q={}, **kw):
        a = RotaryArgs(q=RotarySide(**{**side, **q}), k=RotarySide(**side), **{**good, **kw})
        return lib.sa2_rotary_fwd(C.byref(a)), lib.sa2_rotary_bwd(C.byref(a))

    for kw in (dict(b=0), dict(n=0), dict(freqs=0), dict(q=dict(x=0)), dict(q=dict(y=0)), dict(q=dict(gain=0)), dict(q=dict(heads=0)), dict(q=dict(x=A + 4)),
               dict(q=dict(gain=A + 4)), dict(q=dict(sx=_lib.Strides(640, 130, 64)))):
        assert run(**kw) == (1, 1), kw
    for kw in (dict(d=48), dict(pairs=4), dict(pairs=40), dict(pairs=0), dict(dtype=2), dict(gain_dtype=2), dict(b=1 << 16, n=1 << 16)):
        assert run(**kw) == (2, 2), kw
    a = RotaryArgs(q=RotarySide(**side), k=RotarySide(**side), **{**good, "partial": 0})
    assert lib.sa2_rotary_bwd(C.byref(a)) == 3
    a.partial, a.partial_bytes = A, 16
    assert lib.sa2_rotary_bwd(C.byref(a)) == 3 and lib.sa2_rotary_partial_bytes(C.byref(a)) >= 2 * 64 * 4
    a.q.dy = 0
    assert lib.sa2_rotary_bwd(C.byref(a)) == 1
    assert lib.sa2_rotary_fwd(None) == 1 and lib.sa2_rotary_bwd(None) == 1 and lib.sa2_rotary_partial_bytes(None) == 0


def test_plain_rotation_on_the_cpu():
    """The form that layers take without a GPU: turns compose, and keep every pair's length."""
    torch.manual_seed(0)
    x = torch.randn(1, 6, 2, 64, dtype=torch.float32)
    one = torch.ones(64)
    freqs = sa.rotary_frequencies(64)
    a = rotary._plain(x, x, one, one, freqs, 0, 1e-6)[0]
    assert torch.allclose(a[:, 0], torch.nn.functional.rms_norm(x, (64,), None, 1e-6)[:, 0], atol=1e-6)
    b = rotary._plain(x, x, one, one, freqs, 10 ** 6, 1e-6)[0]
    for t in (a, b):
        length = t[..., :32].square() + t[..., 32:].square()
        assert torch.allclose(length, (y := torch.nn.functional.rms_norm(x, (64,), None, 1e-6))[..., :32].square() + y[..., 32:].square(), atol=1e-5)
    # scores of rows i and j depend on their distance alone
    s = lambda t: torch.einsum("bihd,bjhd->bhij", t, t)
    assert torch.allclose(s(a), s(b), atol=1e-3)


def test_positions_behind_any_table():
    """start + n above 2^63 is no small number."""
    lib = _lib.lib()
    table = dict(positions=A, dpositions=A, position_rows=100)
    good = dict(tokens=A, weight=A, out=A, dout=A, dweight=A, workspace=A, workspace_bytes=1 << 20, rows=12, vocab=9, n=4, dim=8, padding=-1, scale=1.0)
    for kw in (dict(start=2 ** 63 - 1), dict(start=2 ** 63 - 4), dict(start=97), dict(position_rows=-2 ** 63), dict(position_rows=3)):
        a = EmbedArgs(**{**good, **table, **kw})
        assert lib.sa2_embed_fwd(C.byref(a)) == 1 and lib.sa2_embed_bwd(C.byref(a)) == 1
    with pytest.raises(ValueError, match="positions"):
        sa.token_embedding(_cuda(2, 3, dtype=torch.long), _cuda(9, 8), _cuda(5, 8), start=2 ** 63 - 1)


def test_widths_next_to_the_largest_int():
    """Pieces of a row are counted in 32 bits."""
    lib = _lib.lib()
    good = dict(tokens=A, weight=A, out=A, dout=A, dweight=A, workspace=A, workspace_bytes=1 << 62, rows=12, vocab=9, n=4, dim=8, padding=-1, scale=1.0)
    for dim in (2 ** 30 + 1, 2 ** 31 - 128, 2 ** 31 - 1):
        a = EmbedArgs(**{**good, "dim": dim})
        assert lib.sa2_embed_fwd(C.byref(a)) == 2 and lib.sa2_embed_bwd(C.byref(a)) == 2
    with pytest.raises(ValueError, match="2\\^30"):
        sa.token_embedding(_cuda(2, 3, dtype=torch.long), _cuda(1, 2 ** 30 + 8))


def test_gradient_scales_beyond_fp32():
    z, t, i = _cuda(4, 50), _cuda(4, 3), _cuda(4, 3, dtype=torch.long)
    for scale in (1e39, -1e39, math.inf):
        with pytest.raises(ValueError, match="grad_scale"):
            sa.distillation_loss_and_grad(z, t, i, grad_scale=scale)
    good = dict(logits=A, teacher=A, index=A, total=A, dlogits=A, workspace=A, workspace_bytes=1 << 20, rows=3, vocab=9, k=2, temperature=1.0)
    for scale in (math.inf, -math.inf, math.nan):
        assert _lib.lib().sa2_distill_both(C.byref(DistillArgs(**{**good, "grad_scale": scale}))) == 1
