"""Norm and rotation of queries and keys against 64 bits.

Tolerances, with u = 2^-24: the mean of squares and its root cost at most 20 u, the factors and the turn 10 u of the two channels'
magnitudes (a sine or cosine is off by 2 u); 32 u of (|u_a| + |u_b|) cover them.  The result is rounded to its type."""
import math

import pytest
import torch

import simplicial_attention_b200 as sa
from simplicial_attention_b200 import rotary

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _half_step(t):
    return torch.finfo(t.dtype).eps / 2


def _angles(freqs, places):
    """Cosines and sines of whole numbers times 64-bit fractions of a turn, the product modulo a turn in integers."""
    turns = [[(p * f) % 2 ** 64 for f in freqs.tolist()] for p in places.flatten().tolist()]
    turns = [[t - 2 ** 64 if t >= 2 ** 63 else t for t in row] for row in turns]
    a = torch.tensor(turns, dtype=torch.float64, device="cuda") * (2 * math.pi / 2.0 ** 64)
    a = a.view(*places.shape, 1, -1)
    return a.cos(), a.sin()


def _other(x, rotated, interleaved):
    """The other channel of every pair, with the sign it has in the first channel's sum (0 where there is none)."""
    o = torch.zeros_like(x)
    if interleaved:
        o[..., 0:rotated:2], o[..., 1:rotated:2] = -x[..., 1:rotated:2], x[..., 0:rotated:2]
    else:
        o[..., :rotated // 2], o[..., rotated // 2:rotated] = -x[..., rotated // 2:rotated], x[..., :rotated // 2]
    return o


def _spread(t, d, interleaved, rest):
    t = t.repeat_interleave(2, -1) if interleaved else torch.cat((t, t), -1)
    return torch.nn.functional.pad(t, (0, d - t.shape[-1]), value=rest)


def _oracle(x, w, cos, sin, eps, interleaved):
    d, rotated = x.shape[-1], 2 * cos.shape[-1]
    u = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    return u * _spread(cos, d, interleaved, 1.0) + _other(u, rotated, interleaved) * _spread(sin, d, interleaved, 0.0), u


def _check(q, k, gq, gk, freqs, places, eps, interleaved, **how):
    leaves = [t.detach().requires_grad_() for t in (q, k, gq, gk)]
    out = sa.qk_norm_rotary(*leaves, freqs, eps=eps, interleaved=interleaved, **how)
    gen = torch.Generator(device="cuda").manual_seed(9)
    dy = [torch.randn(o.shape, generator=gen, device="cuda").to(o.dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, dy)
    cos, sin = _angles(freqs, places)
    rotated, d = 2 * freqs.numel(), q.shape[-1]
    for s in range(2):
        x, w = (leaves[s].detach().double().requires_grad_(), leaves[2 + s].detach().double().requires_grad_())
        want, u = _oracle(x, w, cos, sin, eps, interleaved)
        assert out[s].is_contiguous() and out[s].dtype == q.dtype
        size = u.abs() + _other(u, rotated, interleaved).abs()
        bound = 32 * U * size + want.abs() * _half_step(q) * (1 + 2 ** -7)
        assert ((out[s].double() - want).abs() <= bound).all()
        e = dy[s].double()
        dx, dw = torch.autograd.grad(want, [x, w], e)
        # e turned back is off by 16 u of its pair's magnitudes, the products and the mean over the head by 32 u of theirs
        hat = u.detach() / w.detach()
        rstd = (x.detach().square().mean(-1, keepdim=True) + eps).rsqrt()
        size = (e.abs() + _other(e, rotated, interleaved).abs()) * w.detach().abs()
        bound = 64 * U * rstd * (size + hat.abs() * (size * hat.abs()).mean(-1, keepdim=True)) + dx.abs() * _half_step(q) * (1 + 2 ** -7)
        assert ((grads[s].double() - dx).abs() <= bound).all()
        terms = (e.abs() + _other(e, rotated, interleaved).abs()) * hat.abs()
        count = terms[..., 0].numel()
        bound = (count + 64) * U * terms.sum((0, 1, 2)) + dw.abs() * _half_step(gq) * (1 + 2 ** -7)
        assert ((grads[2 + s].double() - dw).abs() <= bound).all()
    return out, grads


def _inputs(b, n, hq, hk, d, dtype, gain_dtype=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    packed = torch.randn(b, n, (hq + 2 * hk) * d, generator=gen, device="cuda").to(dtype)
    q, k = packed[..., :hq * d].unflatten(-1, (hq, d)), packed[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    gains = [(1 + 0.3 * torch.randn(d, generator=gen, device="cuda")).to(gain_dtype) for _ in range(2)]
    return q, k, *gains


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("b, n, hq, hk, d, rotated", [
    (1, 1, 1, 1, 32, 16), (2, 3, 3, 1, 32, 32), (3, 41, 8, 4, 64, 64), (1, 130, 5, 5, 64, 48), (2, 67, 4, 2, 128, 128), (1, 33, 6, 3, 128, 64),
    (1, 19, 2, 1, 256, 256), (2, 10, 3, 3, 256, 80), (40, 1, 8, 4, 64, 64), (1, 700, 48, 16, 64, 64),
], ids=str)
def test_against_64_bits(b, n, hq, hk, d, rotated, interleaved, dtype):
    q, k, gq, gk = _inputs(b, n, hq, hk, d, dtype)
    start = 5
    places = (start + torch.arange(n, device="cuda")).expand(b, n)
    _check(q, k, gq, gk, sa.rotary_frequencies(rotated, device="cuda"), places, 1e-6, interleaved, start=start)


@pytest.mark.parametrize("far", [0, 10 ** 6, 2 ** 31 + 5, 2 ** 53 + 1, -7, -2 ** 62])
def test_far_positions_and_a_row_for_each_sequence(far):
    q, k, gq, gk = _inputs(3, 20, 2, 1, 64, torch.float32)
    freqs = sa.rotary_frequencies(64, theta=500000.0, device="cuda")
    places = far + torch.arange(20, device="cuda") + torch.tensor([[0], [300], [11]], device="cuda")
    _check(q, k, gq, gk, freqs, places, 1e-5, False, positions=places)
    one = places[1]
    _check(q, k, gq, gk, freqs, one.expand(3, 20), 1e-5, True, positions=one)
    _check(q, k, gq, gk, freqs, one.expand(3, 20), 1e-5, False, positions=one[None])
    _check(q, k, gq, gk, freqs, places, 1e-5, False, positions=places.t().contiguous().t())
    a, b = (sa.qk_norm_rotary(q, k, gq, gk, freqs, positions=p) for p in (one.expand(3, 20), one))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_frequencies():
    f = sa.rotary_frequencies(64, theta=10000.0)
    assert f.dtype == torch.int64 and f.shape == (32,)
    for i in (0, 1, 17, 31):
        # one rounding of fp64 in the power, one in the quotient, one of the last 64-bit place
        want = 10000.0 ** (-2 * i / 64) / (2 * math.pi)
        assert abs(f[i].item() / 2.0 ** 64 - want) <= 4 * 2.0 ** -53 * want + 2.0 ** -64
    given = torch.tensor([7.0, -1.0, 0.0, 1e-9] * 4, dtype=torch.float64)
    f = sa.rotary_frequencies(32, inv_freq=given)
    turns = given / (2 * math.pi)
    back = f.double() / 2.0 ** 64
    assert ((back - turns) - (back - turns).round()).abs().max() <= 2.0 ** -52
    # far positions against the angle in 64-bit floating point, whose product is good to 2^-52 of itself
    q = torch.ones(1, 1, 1, 64, device="cuda")
    for p in (3, 12345, 10 ** 6):
        out = sa.qk_norm_rotary(q, q, *[torch.ones(64, device="cuda")] * 2, sa.rotary_frequencies(64, device="cuda"), start=p, eps=0.0)[0][0, 0, 0].double().cpu()
        angle = p * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
        want = torch.cat((angle.cos() - angle.sin(), angle.cos() + angle.sin()))
        assert (out - want).abs().max() <= 32 * U * 2 + p * 2.0 ** -50


def test_strides_alignment_and_gain_types():
    gen = torch.Generator(device="cuda").manual_seed(3)
    freqs = sa.rotary_frequencies(64, device="cuda")
    places = torch.arange(11, device="cuda").expand(2, 11)
    heads_first = torch.randn(2, 4, 11, 64, generator=gen, device="cuda").transpose(1, 2)
    odd = torch.randn(2, 11, 3, 67, generator=gen, device="cuda")[..., 3:]                # no row on a 16-byte boundary
    turned = torch.randn(2, 11, 64, 3, generator=gen, device="cuda").transpose(2, 3)       # channels apart
    one = torch.randn(1, 1, 2, 64, generator=gen, device="cuda").expand(2, 11, 2, 64)
    g = [(1 + 0.1 * torch.randn(64, generator=gen, device="cuda")) for _ in range(2)]
    for q, k in ((heads_first, odd), (turned, one), (odd, heads_first)):
        _check(q, k, *g, freqs, places, 1e-6, False)
        _check(q.bfloat16(), k.bfloat16(), *[t.bfloat16() for t in g], freqs, places, 1e-6, True)
    far = torch.randn(129, generator=gen, device="cuda")[1:]
    _check(heads_first, odd, far[:64], far[64:], freqs, places, 1e-6, False)
    gap = torch.randn(7, 11, 2, 64, generator=gen, device="cuda")[3:4]
    _check(gap, gap, *g, freqs, places[:1], 1e-6, False)


def test_default_eps_zeros_and_empty():
    q, k, gq, gk = _inputs(1, 5, 2, 1, 64, torch.bfloat16)
    q = q.clone()
    q[0, 2] = 0                          # a head of zeros stays zeros
    freqs = sa.rotary_frequencies(64, device="cuda")
    out, _ = _check(q, k, gq, gk, freqs, torch.arange(5, device="cuda")[None], 2.0 ** -7, False)
    again = sa.qk_norm_rotary(q, k, gq, gk, freqs)
    assert torch.equal(out[0], again[0]) and (again[0][0, 2] == 0).all()
    leaves = [t.detach().requires_grad_() for t in (q[:, :0], k[:, :0], gq, gk)]
    out = sa.qk_norm_rotary(*leaves, freqs)
    assert out[0].shape == (1, 0, 2, 64)
    grads = torch.autograd.grad(out, leaves, [torch.zeros_like(o) for o in out])
    assert (grads[2] == 0).all() and (grads[3] == 0).all()


def test_gradient_against_differences():
    """A step to either side along a direction.  The operator's own roundings (bounds above, over the step) and what the step misses, taken
    from the oracle in 64 bits, are what the difference may be off by."""
    q, k, gq, gk = _inputs(2, 9, 3, 2, 64, torch.float32)
    freqs = sa.rotary_frequencies(64, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    leaves = [t.detach().contiguous().requires_grad_() for t in (q, k, gq, gk)]
    way = [torch.randn(t.shape, generator=gen, device="cuda") for t in leaves]
    w = [torch.randn(t.shape, generator=gen, device="cuda") for t in (q, k)]
    h = 2.0 ** -8
    cos, sin = _angles(freqs, torch.arange(9, device="cuda").expand(2, 9))

    def kernel(ts):
        return sum((o.double() * v.double()).sum() for o, v in zip(sa.qk_norm_rotary(*ts, freqs, eps=1e-6), w))

    def oracle(ts):
        return sum((_oracle(ts[s].double(), ts[2 + s].double(), cos, sin, 1e-6, False)[0] * w[s].double()).sum() for s in range(2))

    grads = torch.autograd.grad(kernel(leaves), leaves)
    slope = sum((g.double() * v.double()).sum() for g, v in zip(grads, way))
    sides = [[(t + s * h * v).detach() for t, v in zip(leaves, way)] for s in (1, -1)]
    apart = (kernel(sides[0]) - kernel(sides[1])) / (2 * h)
    true = torch.autograd.grad(oracle(leaves), leaves)
    missed = ((oracle(sides[0]) - oracle(sides[1])) / (2 * h) - sum((g.double() * v.double()).sum() for g, v in zip(true, way))).abs()
    outs = sa.qk_norm_rotary(*leaves, freqs, eps=1e-6)
    rounding = sum((100 * U * o.abs().double() * v.abs().double()).sum() + (100 * U * v.abs().double()).sum() for o, v in zip(outs, w)) / h
    assert (apart - slope).abs() <= missed + rounding
    assert missed + rounding <= 0.02 * sum(g.double().norm() * v.double().norm() for g, v in zip(grads, way))       # (it says something)


def test_same_bits_streams_and_captured():
    q, k, gq, gk = _inputs(4, 333, 8, 4, 64, torch.bfloat16, torch.bfloat16)
    freqs = sa.rotary_frequencies(64, device="cuda")
    leaves = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (q, k, gq, gk)]
    dy = [torch.randn_like(leaves[0]), torch.randn_like(leaves[1])]
    positions = torch.randint(0, 5000, (4, 333), device="cuda")

    def step():
        out = sa.qk_norm_rotary(*leaves, freqs, positions=positions)
        grads = torch.autograd.grad(out, leaves, dy)
        return [*(o.detach() for o in out), *grads]          # (no graph outlives the call)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    positions.random_(0, 100000)
    graph.replay()
    for a, b in zip(res, step()):
        assert torch.equal(a, b)


def test_one_side_used_and_no_second_backward():
    q, k, gq, gk = _inputs(1, 7, 2, 1, 64, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (q, k, gq, gk)]
    freqs = sa.rotary_frequencies(64, device="cuda")
    out = sa.qk_norm_rotary(*leaves, freqs)
    grads = torch.autograd.grad(out[0].sum(), leaves, retain_graph=True)
    assert (grads[1] == 0).all() and (grads[3] == 0).all() and (grads[0] != 0).any()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out[0].sum(), leaves, create_graph=True)


def test_plain_form_agrees():
    q, k, gq, gk = _inputs(2, 30, 3, 1, 64, torch.float32)
    for il in (False, True):
        freqs = sa.rotary_frequencies(48, device="cuda")
        a = sa.qk_norm_rotary(q, k, gq, gk, freqs, start=77, eps=1e-6, interleaved=il)
        b = rotary._plain(q, k, gq, gk, freqs, 77, 1e-6, il)
        for x, y in zip(a, b):
            assert (x - y).abs().max() <= 100 * U * y.abs().max()
