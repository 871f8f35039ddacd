"""Sampled tokens against the definition in 64 bits, token for token; the inputs' random numbers come from fixed seeds, so that none lies
within the 2^-46 of a border that the kernel's whole-number masses allow."""
import math

import numpy as np
import pytest
import torch

import simplicial_attention_b200 as sa

pytestmark = pytest.mark.gpu


def _value(setting, r):
    return None if setting is None else (setting[r].item() if isinstance(setting, torch.Tensor) else setting)


def _oracle(logits, uniform, temperature=1.0, top_k=None, top_p=None, min_p=None):
    tokens, logprobs = [], []
    for r, z in enumerate(logits.double().cpu()):
        if z.isnan().any() or z.max().isinf():
            tokens.append(-1)
            logprobs.append(float("nan"))
            continue
        t, k, p, m = (_value(s, r) for s in (temperature, top_k, top_p, min_p))
        order = torch.argsort(-z, stable=True)
        if t == 0:
            tokens.append(order[0].item())
            logprobs.append(0.0)
            continue
        x = (z - z.max()) / t
        w = x.exp()
        count = z.numel() if k is None or k <= 0 else min(k, z.numel())
        if p is not None and p < 1:
            mass = w[order[:count]].cumsum(0)
            count = min(count, 1 + int((mass < p * mass[-1]).sum()))
        keep = torch.zeros_like(w, dtype=torch.bool)
        keep[order[:max(1, count)]] = True
        if m is not None and m > 0:
            keep &= (w >= min(m, 1.0))
        mass = (w * keep).cumsum(0)
        u = uniform.flatten()[r].item()
        j = min(int((mass <= u * mass[-1]).sum()), int(keep.nonzero().max()))
        tokens.append(j)
        logprobs.append((x[j] - mass[-1].log()).item())
    return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)


def _check(logits, uniform, **settings):
    token, logprob = sa.sample_tokens(logits, uniform, return_logprobs=True, **settings)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32 and token.shape == logits.shape[:-1]
    flat = {k: v.flatten() if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
    want, want_log = _oracle(logits.flatten(0, -2) if logits.dim() > 1 else logits[None], uniform, **flat)
    assert torch.equal(token.flatten().cpu(), want)
    bad = want_log.isnan()
    assert torch.equal(logprob.flatten().cpu().isnan(), bad)
    # one rounding to fp32, and the masses' 2^-40 at most
    assert ((logprob.flatten().cpu().double() - want_log).abs() <= want_log.abs() * 2.0 ** -24 + 1e-9)[~bad].all()
    return token


def _logits(rows, vocab, dtype, seed=0, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen, device="cuda") * spread).to(dtype), torch.rand(rows, generator=gen, device="cuda")


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=50, top_p=0.95),
            dict(temperature=1.3, top_k=200, top_p=0.8, min_p=0.02), dict(temperature=0.0), dict(top_p=1e-6), dict(min_p=1.0), dict(top_k=10 ** 9, top_p=1.0, min_p=0.0),
            dict(temperature=1e-4), dict(temperature=0.0, top_p=0.5, min_p=0.5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: " ".join(f"{k}={v}" for k, v in s.items()) or "none")
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (7, 31), (40, 256), (9, 4097), (30, 9001)], ids=str)
def test_against_the_definition(rows, vocab, settings, dtype):
    _check(*_logits(rows, vocab, dtype), **settings)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab", [(1, 32000), (100, 50001), (2, 131072), (40, 128000), (1, 500001), (1, 1000003)], ids=str)
def test_several_ctas_a_row(rows, vocab, dtype):
    z, u = _logits(rows, vocab, dtype)
    for settings in (dict(), dict(top_k=64), dict(top_p=0.9, min_p=0.001), dict(top_k=5000, top_p=0.99, temperature=0.8)):
        _check(z, u, **settings)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab", [(300, 100), (260, 129), (400, 1000), (170, 16384)], ids=str)
def test_many_short_rows(rows, vocab, dtype):
    """More rows than SMs: CTAs of 128 threads."""
    z, u = _logits(rows, vocab, dtype)
    for settings in (dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=300, top_p=0.99, temperature=1.7), dict(temperature=0.0)):
        _check(z, u, **settings)


def test_more_rows_than_fit_and_rows_from_memory():
    """200 rows of 128001: a CTA a row, which does not fit into shared memory and, odd, begins on no 16-byte boundary; then such that do."""
    for vocab in (128001, 60000):
        z, u = _logits(200, vocab, torch.float32)
        few = slice(0, 200, 19)                          # (the oracle is slow)
        for settings in (dict(top_p=0.6), dict(top_k=2000, top_p=0.9), dict(min_p=0.02, top_p=0.9), dict()):
            got = sa.sample_tokens(z, u, **settings)
            assert torch.equal(got[few].cpu(), _oracle(z[few], u[few], **settings)[0])


@pytest.mark.parametrize("vocab", [60, 5000, 70000])
def test_extreme_temperatures_and_logits(vocab):
    z, u = _logits(6, vocab, torch.float32)
    for t in (1e-30, 1e-7, 1e-3, 30.0, 1e6, 1e30, 1e300):
        for settings in (dict(temperature=t), dict(temperature=t, top_k=9), dict(temperature=t, top_p=0.7), dict(temperature=t, min_p=0.3, top_p=0.9)):
            _check(z, u, **settings)
    far = z.clone()
    far[0] += 1e6
    far[1] *= 1e30
    far[2] = -3.4e38
    far[2, :3] = -3.3e38
    far[3] = torch.finfo(torch.float32).min
    far[3, 5:] = float("-inf")
    far[4] *= 1e-42                          # subnormal numbers
    far[5] = 0.0
    far[5, 7] = 1e-45
    for t in (1e-40, 1.0, 1e37):
        for settings in (dict(temperature=t), dict(temperature=t, top_k=4), dict(temperature=t, top_p=0.8), dict(temperature=t, min_p=0.5)):
            _check(far, u, **settings)


@pytest.mark.parametrize("offset", [0.0, 64.0, 3000.0, -500.0])
def test_cuts_among_five_hundred(offset):
    """Around the most logits that are sorted at once, with numbers far apart and equal ones on both sides."""
    z, u = _logits(8, 30000, torch.float32)
    z = z + offset
    for dtype in (torch.float32, torch.bfloat16):
        for k in (350, 500, 511, 512, 513, 600):
            _check(z.to(dtype), u, top_k=k)
            _check(z.to(dtype), u, top_k=k, top_p=0.97, temperature=2.0)
        for p in (0.3, 0.45, 0.6):
            _check(z.to(dtype), u, top_p=p)


@pytest.mark.parametrize("vocab", [50, 3000, 40001])
def test_equal_logits_rank_by_index(vocab):
    z = torch.zeros(6, vocab, device="cuda")
    z[1, vocab // 2:] = 1.0
    z[2, ::3] = -0.0                         # equal to 0
    z[3, 1::2] = float("-inf")
    z[4, :] = -5.0
    z[5, 7] = 3.0
    u = torch.tensor([0.0, 0.5, 0.999999, 0.3, 0.77, 0.9999], device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        for settings in (dict(), dict(top_k=3), dict(top_k=vocab // 2 + 5), dict(top_p=0.25), dict(top_k=20, top_p=0.5), dict(min_p=1.0), dict(temperature=0.0)):
            _check(z.to(dtype), u, **settings)
    coarse, u = _logits(20, vocab, torch.float32)
    for settings in (dict(top_k=7), dict(top_p=0.5), dict(top_k=100, top_p=0.7, min_p=0.1)):
        _check(coarse.round(), u, **settings)            # many ties at the cut


@pytest.mark.parametrize("vocab", [64, 2000, 70001])
def test_rows_without_a_distribution(vocab):
    z, u = _logits(8, vocab, torch.float32)
    z[0] = float("-inf")
    z[1, 5] = float("nan")
    z[2, vocab - 1] = float("inf")
    z[3, :-1] = float("-inf")                # one token is left
    z[4, 1:] = torch.finfo(torch.float32).min
    z[5, ::2] = float("-inf")
    z[6] = torch.finfo(torch.float32).min    # all equally unlikely
    for settings in (dict(), dict(top_k=5), dict(top_p=0.9, min_p=0.1), dict(temperature=0.0)):
        token = _check(z, u, **settings)
        assert token[:3].tolist() == [-1, -1, -1] and token[3] == vocab - 1 and token[4] == 0


def test_settings_for_each_row():
    z, u = _logits(12, 5000, torch.bfloat16)
    t = torch.linspace(0.0, 2.0, 12, device="cuda")
    k = torch.tensor([0, 1, 2, 5, 10, 50, 100, 1000, 4999, 5000, 6000, -3], device="cuda")
    p = torch.linspace(0.05, 1.2, 12, device="cuda")
    m = torch.linspace(0.0, 0.4, 12, device="cuda").flip(0)
    together = _check(z, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert torch.equal(together, sa.sample_tokens(z, u, temperature=t.double(), top_k=k.int(), top_p=p, min_p=m))
    for r in range(12):                      # a row does not depend on the rows beside it
        alone = sa.sample_tokens(z[r], u[r], temperature=t[r].item(), top_k=k[r].item(), top_p=p[r].item(), min_p=m[r].item())
        assert alone.shape == () and alone == together[r]


def test_strided_rows_shapes_and_numbers():
    gen = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(3, 5, 777, generator=gen, device="cuda") * 2
    u = torch.rand(3, 5, generator=gen, device="cuda")
    a = _check(z, u, top_k=30)
    assert a.shape == (3, 5)
    assert torch.equal(a[:, -1], sa.sample_tokens(z[:, -1], u[:, -1], top_k=30))
    assert torch.equal(a, sa.sample_tokens(z.transpose(0, 2).contiguous().transpose(0, 2), u.double(), top_k=30))
    odd = torch.randn(4, 1001, generator=gen, device="cuda").bfloat16()[:, 3:]
    _check(odd, u[0, :4], top_p=0.8)
    # the ends of [0, 1), and beyond
    one = z[0, :1].expand(6, 777)
    ends = torch.tensor([0.0, 1 - 2.0 ** -53, 2.0 ** -60, 1.0, -1.0, 2.0], dtype=torch.float64, device="cuda")
    got = sa.sample_tokens(one, ends, top_k=30)
    kept = one[0].topk(30).indices
    assert got[0] == got[2] == got[4] == kept.min() and got[1] == got[3] == got[5] == kept.max()


def test_frequencies_follow_the_distribution():
    z = torch.tensor([2.0, 0.0, 1.0, -1.0, float("-inf"), 0.5], device="cuda")
    n = 200000
    gen = torch.Generator(device="cuda").manual_seed(8)
    tokens = sa.sample_tokens(z.expand(n, 6), torch.rand(n, generator=gen, device="cuda"), temperature=0.8, top_k=4)
    w = torch.exp(z / 0.8)
    w[3] = 0
    want = w / w.sum()
    got = torch.bincount(tokens, minlength=6) / n
    assert got[3] == 0 and got[4] == 0
    assert (got - want).abs().max() <= 5 * 0.5 / n ** 0.5            # five standard deviations


def test_nothing_streams_and_captured():
    assert sa.sample_tokens(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)
    z, u = _logits(5, 40000, torch.float32)
    first = sa.sample_tokens(z, u, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(first, sa.sample_tokens(z, u, top_p=0.9))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = sa.sample_tokens(z, u, top_p=0.9, top_k=1000, return_logprobs=True)
    for seed in (1, 2):
        other = _logits(5, 40000, torch.float32, seed=seed)
        z.copy_(other[0])
        u.copy_(other[1])
        graph.replay()
        want = sa.sample_tokens(z, u, top_p=0.9, top_k=1000, return_logprobs=True)
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 5000, 140000])
def test_floor_at_a_logit_of_zero(vocab, dtype):
    """best + T log(min_p) cancels: the floor lies among the smallest numbers of the type.  Logits stay clear of the floor, whose last bits
    are a matter of rounding."""
    z, u = _logits(4, vocab, dtype)
    z = torch.where(z.abs() < 1e-3, torch.full_like(z, 0.5), z).clamp(max=0.75)
    for best, temperature, min_p in ((5.0, 1.0, math.exp(-5)), (1.0, 1 / math.log(2), 0.5), (7.0, 0.7, math.exp(-10))):
        z[:, 17] = best
        for settings in (dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=200, top_p=0.99)):
            _check(z, u, temperature=temperature, min_p=min_p, **settings)


def _tokens_of_long_sums(logits, uniform, temperature, top_k=None, top_p=None, min_p=None):
    """As _oracle, with sums of 64-bit significands.  A thousand equal logits and two thousand of a weight of 4e-14 have 1000 + 8.7e-11, which
    a sum in fp64 takes for 1000; the 701st token stays for a top_p of 0.7 all the same: 700 is less than 0.7 (1000 + 8.7e-11)."""
    tokens = []
    for r, z in enumerate(logits.double().cpu().numpy()):
        if np.isnan(z).any() or np.isinf(z.max()):
            tokens.append(-1)
            continue
        w = np.exp(((z - z.max()) / temperature).astype(np.longdouble))
        order = np.lexsort((np.arange(z.size), -z))
        count = z.size if top_k is None else min(top_k, z.size)
        if top_p is not None:
            mass = w[order[:count]].cumsum()
            count = min(count, 1 + int((mass < np.longdouble(top_p) * mass[-1]).sum()))
        keep = np.zeros(z.size, dtype=bool)
        keep[order[:count]] = True
        if min_p is not None:
            keep &= w >= min_p
        mass = (w * keep).cumsum()
        tokens.append(min(int((mass <= np.longdouble(uniform[r].item()) * mass[-1]).sum()), int(keep.nonzero()[0].max())))
    return tokens


@pytest.mark.parametrize("vocab", [200, 3000, 70000])
def test_rows_that_span_more_than_fp32(vocab):
    """best - v is no fp32 number, and at these temperatures v has a mass all the same."""
    _, u = _logits(4, vocab, torch.float32)
    z = torch.full((4, vocab), -3e38, device="cuda")
    z[0, ::2] = 3e38
    z[1] = torch.linspace(-3.3e38, 3.3e38, vocab, device="cuda")
    z[2, 1::2] = torch.finfo(torch.float32).max
    z[2, ::2] = torch.finfo(torch.float32).min
    z[3, : vocab // 3] = 1e38
    for t in (3e36, 9e36, 1e37, 1.3e37, 1e38, 3e38):
        for settings in (dict(), dict(top_k=vocab * 5 // 7), dict(top_k=vocab // 3), dict(top_p=0.9999), dict(top_p=0.7), dict(top_k=vocab * 5 // 7, top_p=0.95), dict(min_p=0.01),
                         dict(min_p=0.001, top_p=0.99)):
            for x in (z, z[:1].bfloat16()):
                assert sa.sample_tokens(x, u[:x.shape[0]], temperature=t, **settings).tolist() == _tokens_of_long_sums(x, u, t, **settings)
