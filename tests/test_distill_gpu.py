"""Distillation from a teacher's top logits against 64 bits.

Tolerances, with u = 2^-24: a weight 2^x is off by 4 u (ex2) and by 2 u |x| (its exponent's roundings), the sum of a row by at most
(vocab / 32 + 64) u more, the logarithm and the probabilities by the same.  `slack` below is the sum of these; results are rounded to
their types."""
import math

import pytest
import torch

import simplicial_attention_b200 as sa

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _half_step(t):
    return torch.finfo(t.dtype).eps / 2


def _inputs(rows, vocab, k, dtype, teacher_dtype=torch.float32, seed=0, spread=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(rows, vocab, generator=gen, device="cuda") * spread).to(dtype)
    t = (torch.randn(rows, k, generator=gen, device="cuda") * spread).to(teacher_dtype)
    i = torch.rand(rows, vocab, generator=gen, device="cuda").argsort(-1)[:, :k]
    if k > vocab:
        i = torch.randint(vocab, (rows, k), generator=gen, device="cuda")
    return z, t, i.contiguous()


def _oracle(z, t, i, temperature):
    """Loss of every row, its gradient, whether the row counts."""
    zd = z.double() / temperature
    there = (i >= 0) & (i < z.shape[-1])
    td = (t.double() / temperature).masked_fill(~there, float("-inf"))
    counted = (td > float("-inf")).any(-1)
    p = torch.where(counted[:, None], torch.softmax(td, -1), torch.zeros_like(td))
    place = i.long().clamp(0, z.shape[-1] - 1)
    log_q = torch.log_softmax(zd, -1)
    terms = torch.where(p > 0, torch.special.xlogy(p, p) - p * log_q.gather(-1, place), torch.zeros_like(p))
    q = log_q.exp()
    grad = torch.where(counted[:, None], q, torch.zeros_like(q)).scatter_add(-1, place, -p)
    return terms.sum(-1) * temperature ** 2, grad * temperature, counted, q, torch.zeros_like(q).scatter_add(-1, place, p), (p * log_q.gather(-1, place).abs().nan_to_num(0, 0, 0)).sum(-1)


def _check(z, t, i, temperature=1.0, reduction="mean", both=True):
    vocab = z.shape[-1]
    loss_rows, dz, counted, q, p, size = _oracle(z.detach(), t, i, temperature)
    x = (z.double() / temperature - (z.double() / temperature).amax(-1, keepdim=True)).nan_to_num(0, 0, 0).abs() * 1.4427
    far = x.clamp_max(60).amax(-1)                     # (2^-60 and less is nothing)
    slack = 4 * U + 2 * U * far + (vocab / 32 + 64) * U
    rows = max(1, int(counted.sum()))
    divisor = rows if reduction == "mean" else 1
    leaf = z.detach().requires_grad_()
    loss = sa.distillation_loss(leaf, t, i, temperature=temperature, reduction=reduction)
    assert loss.dtype == torch.float32
    per_row = temperature ** 2 * slack * (1 + 0 * size) + 4 * U * (loss_rows.abs() + temperature ** 2 * size)
    per_row = torch.where(counted, per_row, torch.zeros_like(per_row))
    want = loss_rows if reduction == "none" else loss_rows.sum() / divisor
    bound = per_row if reduction == "none" else per_row.sum() / divisor + 2 * U * want.abs()
    # (an exact loss above the largest fp32 number rounds to inf: 2.4e39 where a teacher has a half of its mass on the lowest bf16 value, T = 100)
    over = want.abs() > torch.finfo(torch.float32).max
    assert (loss[over] == float("inf")).all() and ((loss.double() - want).abs() <= bound)[~over].all()

    gen = torch.Generator(device="cuda").manual_seed(5)
    gout = torch.rand(loss.shape, generator=gen, device="cuda") + 0.5
    got = torch.autograd.grad(loss, leaf, gout)[0]
    assert got.dtype == z.dtype and got.shape == z.shape
    if reduction != "none":
        gout = gout.expand(z.shape[0])

    def grad_close(got, g):
        g = g.double()[:, None] / divisor
        # (a weight below 2^-126 of the largest is flushed to 0 by ex2.ftz, and the sum of a row is at least 1: q is off by 2^-126 at most)
        bound = g.abs() * temperature * (q * (2 * slack + 2 * U * x + 8 * U)[...] + p * 1032 * U + 2.0 ** -126) + (dz * g).abs() * _half_step(z) * (1 + 2 ** -7) + 2.0 ** -133
        assert ((got.double() - dz * g).abs() <= bound).all()

    slack = slack[:, None]
    grad_close(got, gout)
    assert (got[~counted] == 0).all()
    if both and reduction != "none":
        one, grad = sa.distillation_loss_and_grad(z.detach(), t, i, temperature=temperature, reduction=reduction, grad_scale=3.0)
        assert (one[over] == float("inf")).all() and ((one.double() - want).abs() <= bound)[~over].all()
        grad_close(grad, torch.full_like(gout, 3.0))
        assert (grad[~counted] == 0).all()
    return loss, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab, k, temperature", [
    (1, 1, 1, 1.0), (3, 2, 5, 0.5), (17, 7, 3, 2.0), (9, 256, 8, 1.0), (33, 255, 16, 1.5), (8, 2048, 64, 1.0), (5, 2049, 64, 3.0), (70, 4097, 33, 1.0),
    (3, 32000, 100, 2.0), (2, 50257 + 1, 1024, 1.0), (1, 131071, 1, 0.7), (4, 128000, 64, 2.0), (2, 262145, 20, 1.0), (1, 700001, 9, 4.0),
], ids=str)
def test_against_64_bits(rows, vocab, k, temperature, dtype):
    z, t, i = _inputs(rows, vocab, k, dtype)
    _check(z, t, i, temperature)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("vocab", [300, 5003, 40000])
def test_reductions_and_absent_entries(reduction, vocab):
    z, t, i = _inputs(13, vocab, 12, torch.float32, torch.bfloat16)
    i[2] = -1                                # no teacher
    i[5, 3:] = -1
    t[5, 3:] = float("nan")                  # ... whatever stands there
    i[6, ::2] = vocab + 7
    i[7, 1:] = i[7, 0]                       # one token alone
    i[8, 6:] = i[8, :6]                      # tokens twice
    t[9, 4:] = float("-inf")
    t[10] = float("-inf")                    # no mass
    t[11, 2] = torch.finfo(torch.bfloat16).min
    i[12, 1:] = -5
    i[12, 0] = vocab - 1
    _check(z, t, i, 1.7, reduction)
    _check(z, t, i.int(), 1.7, reduction)
    _check(z[:3], t[10:11].expand(3, 12), i[:3], 1.0, reduction)             # no row counts


@pytest.mark.parametrize("k", [2, 31, 32, 33, 64, 257, 512, 513, 1024])
@pytest.mark.parametrize("vocab", [1030, 140000])
def test_entries_of_one_token(vocab, k):
    z, t, i = _inputs(6, vocab, k, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(k)
    i[0] = vocab - 1                         # all the same
    i[1] = torch.arange(k, device="cuda").flip(0) // 2
    i[2] = torch.randint(max(1, k // 3), (k,), generator=gen, device="cuda") * (vocab // max(1, k // 3))
    i[3] = (torch.arange(k, device="cuda") * 65536) % vocab
    i[4, ::2] = -1
    i[4, 1::2] = 5
    i[5, -1] = i[5, 0]
    _check(z, t, i, 1.0)
    _check(z, t, i, 1.0, "none")


@pytest.mark.parametrize("temperature", [0.01, 1.0, 100.0])
@pytest.mark.parametrize("vocab", [300, 5001, 60000])
def test_bf16_logits_far_from_zero(vocab, temperature):
    z, t, i = _inputs(8, vocab, 7, torch.bfloat16)
    z[0] += 30000
    z[1] -= 30000
    z[2] = 20000 * z[2]
    z[3] = 128 * z[3].round() + 32768        # neighbouring values of the type
    z[4, : vocab // 2] = torch.finfo(torch.bfloat16).min
    z[5] = torch.finfo(torch.bfloat16).min
    z[6, ::3] = float("-inf")
    z[6, i[6]] = 1.0
    z[7] = torch.linspace(-900, 900, vocab, device="cuda").bfloat16()       # the maximum moves all the way
    _check(z, t, i, temperature)


@pytest.mark.parametrize("vocab", [64, 3001, 90000])
def test_masked_students(vocab):
    z, t, i = _inputs(6, vocab, 5, torch.float32)
    i = (torch.arange(5, device="cuda") * 3 + torch.arange(6, device="cuda")[:, None]).contiguous()
    z[0, 40:] = float("-inf")                # tokens that are out of the question
    z[1, 41:] = torch.finfo(torch.float32).min
    z[2] = 1e4 * z[2]
    z[3] = z[3] + 3e4
    z[4] = 0.0
    _check(z, t, i, 2.0, "none")
    _check(z, t, i, 2.0, "mean")
    # the teacher wants what the student rules out
    z[0, i[0, 0]] = float("-inf")
    assert sa.distillation_loss(z, t, i, reduction="none")[0] == float("inf")
    # NaN stays in its row
    z[5, 63] = float("nan")
    loss = sa.distillation_loss(z, t, i, reduction="none")
    assert loss[5].isnan() and not loss[1:5].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [100, 2500, 60001])
def test_strided_rows_and_shapes(vocab, dtype):
    z, t, i = _inputs(6, vocab + 3, 4, dtype)
    i.clamp_(max=vocab - 1)
    i[:, 1:] = torch.where(i[:, 1:] == i[:, :1], torch.full_like(i[:, 1:], -1), i[:, 1:])
    for view in (z[:, 1:vocab + 1], z[:, 3:], z[::2, :vocab], z[:, :vocab].t().contiguous().t()):
        m = view.shape[0]
        _check(view, t[:m], i[:m], 1.0)
    _check(z[:, :vocab], torch.cat((t, t), 1)[:, 1:5], torch.cat((i, i), 1)[:, 1:5], 1.0)
    three = z.view(2, 3, -1)[..., :vocab]
    leaf = three.detach().requires_grad_()
    a = sa.distillation_loss(leaf, t.view(2, 3, 4), i.view(2, 3, 4), reduction="none")
    assert a.shape == (2, 3)
    # the order of a row's sum follows its 16-byte boundaries: both are within the bound of _check, whose exponents stay below 60 here
    packed = sa.distillation_loss(z[:, :vocab].contiguous(), t, i, reduction="none")
    assert ((a.flatten() - packed).abs() <= 2 * ((4 + 2 * 60 + vocab / 32 + 64) * U + 4 * U * (packed.abs() + 60))).all()
    grad = torch.autograd.grad(a.sum(), leaf)[0]
    assert grad.shape == three.shape
    one, g = sa.distillation_loss_and_grad(three, t.view(2, 3, 4), i.view(2, 3, 4), reduction="sum")
    assert one.shape == () and g.shape == three.shape
    # one row without a batch
    assert torch.equal(sa.distillation_loss(three[1, 2], t[5], i[5], reduction="none"), a[1, 2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,first,count", [(5, 0, 1), (5, 4, 1), (50, 8, 8), (4097, 800, 8), (4097, 0, 4097)])
def test_nan_anywhere_shows(vocab, first, count, dtype):
    z, t, i = _inputs(3, vocab, 4, dtype)
    clean = sa.distillation_loss(z, t, i, reduction="none")
    z[1, first:first + count] = float("nan")
    leaf = z.clone().requires_grad_()
    loss = sa.distillation_loss(leaf, t, i, reduction="none")
    loss.sum().backward()
    assert loss[1].isnan() and torch.equal(loss[::2], clean[::2])
    assert leaf.grad[1].isnan().all() and not leaf.grad[::2].isnan().any()
    total, grad = sa.distillation_loss_and_grad(z, t, i)
    assert total.isnan() and grad[1].isnan().all() and not grad[::2].isnan().any()


@pytest.mark.parametrize("temperature", [1e-30, 1e-8, 1e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [300, 4099])
def test_lowest_values_and_temperatures_far_from_one(vocab, dtype, temperature):
    z = torch.full((2, vocab), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    z[:, 7], z[0, 9] = 2.0, 2.0
    t, i = torch.tensor([[1.0, 1.0], [3.0, 3.0]], device="cuda"), torch.tensor([[7, 9], [7, 7]], device="cuda")
    _, dz, *_ = _oracle(z, t, i, float(torch.tensor(temperature, dtype=torch.float32)))
    leaf = z.requires_grad_()
    both = sa.distillation_loss_and_grad(z.detach(), t, i, reduction="sum", temperature=temperature)[1]
    grad = torch.autograd.grad(sa.distillation_loss(leaf, t, i, reduction="sum", temperature=temperature), leaf)[0]
    # exponents of the lowest value at T = 1e38 are off by their rounding, 2^-23 of 4.9; the sum of a row and its inverse as above
    bound = temperature * ((vocab / 32 + 100) * U + 1.0 / vocab * _half_step(z)) + dz.abs() * _half_step(z) + 2.0 ** -133
    assert ((grad.double() - dz).abs() <= bound).all() and ((both.double() - dz).abs() <= bound).all()


def test_mean_over_many_rows():
    z, t, i = _inputs(20000, 2100, 2, torch.bfloat16)
    i[::3] = -1
    loss, grad = sa.distillation_loss_and_grad(z, t, i)
    rows = sa.distillation_loss(z, t, i, reduction="none").double()
    counted = 20000 - len(range(0, 20000, 3))
    want = rows.sum() / counted
    assert (loss.double() - want).abs() <= want.abs() * 2 * U
    leaf = z.requires_grad_()
    assert torch.equal(torch.autograd.grad(sa.distillation_loss(leaf, t, i), leaf)[0], grad)
    assert (grad[::3] == 0).all() and (grad[1::3] != 0).any()


def test_nothing():
    z, t, i = torch.zeros(0, 7, device="cuda"), torch.zeros(0, 2, device="cuda"), torch.zeros(0, 2, dtype=torch.long, device="cuda")
    leaf = z.requires_grad_()
    loss = sa.distillation_loss(leaf, t, i)
    assert loss == 0 and torch.autograd.grad(loss, leaf)[0].shape == (0, 7)
    loss, grad = sa.distillation_loss_and_grad(z.detach(), t, i)
    assert loss == 0 and grad.shape == (0, 7)


def test_gradient_against_differences():
    """A step to either side along a direction; what the step misses comes from the oracle, roundings are bounded as above."""
    z, t, i = _inputs(5, 900, 6, torch.float32)
    leaf = z.requires_grad_()
    loss, grad = _check(z, t, i, 1.3, "sum")
    gen = torch.Generator(device="cuda").manual_seed(6)
    way = torch.randn(z.shape, generator=gen, device="cuda")
    h = 2.0 ** -6
    sides = [(leaf.detach() + s * h * way) for s in (1, -1)]
    loss = sa.distillation_loss(leaf, t, i, temperature=1.3, reduction="sum")
    slope = (torch.autograd.grad(loss, leaf)[0].double() * way.double()).sum()
    apart = [sa.distillation_loss(x, t, i, temperature=1.3, reduction="none").double().sum() for x in sides]
    exact = [_oracle(x, t, i, 1.3)[0].sum() for x in sides]
    true = (_oracle(leaf.detach(), t, i, 1.3)[1] * way.double()).sum()
    missed = ((exact[0] - exact[1]) / (2 * h) - true).abs()
    rounding = 5 * 1.3 ** 2 * (4 + 2 * 40 + 900 / 32 + 64 + 100) * U / h
    assert ((apart[0] - apart[1]) / (2 * h) - slope).abs() <= missed + rounding
    assert missed + rounding <= 0.05 * grad.double().norm() * way.double().norm()


@pytest.mark.parametrize("vocab", [256, 20000])
def test_same_bits_streams_and_captured(vocab):
    z, t, i = _inputs(300, vocab, 16, torch.bfloat16)
    leaf = z.detach().clone().requires_grad_()

    def step():
        loss = sa.distillation_loss(leaf, t, i, temperature=2.0)
        return [loss.detach(), *torch.autograd.grad(loss, leaf), *sa.distillation_loss_and_grad(leaf.detach(), t, i, temperature=2.0)]

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
    with torch.no_grad():
        t.normal_()
        leaf.normal_()
    i.random_(0, vocab)
    graph.replay()
    for a, b in zip(res, step()):
        assert torch.equal(a, b)


def test_the_loss_is_the_callers_and_no_second_backward():
    z, t, i = _inputs(4, 100, 3, torch.float32)
    leaf = z.requires_grad_()
    loss = sa.distillation_loss(leaf, t, i)
    want = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
    loss.data.zero_()
    assert torch.equal(torch.autograd.grad(loss, leaf, retain_graph=True)[0], want)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(loss, leaf, create_graph=True)


@pytest.mark.parametrize("vocab", [300, 5001])
@pytest.mark.parametrize("asked", ["row_loss", "total", "both"])
@pytest.mark.parametrize("forward, backward", [(0, 0), (0, 1), (1, 0), (1, 1)], ids=str)
def test_c_calls_in_any_order(vocab, asked, forward, backward):
    """The gradient of a sum (0) or a mean (1), whatever loss the forward was asked for, from a workspace that held something else."""
    import ctypes as C

    from simplicial_attention_b200 import _lib
    from test_operator_refusals import DistillArgs
    z, t, i = _inputs(70, vocab, 5, torch.float32)
    i[::3] = -1
    lib = _lib.lib()
    lib.sa2_distill_workspace_bytes.restype = C.c_size_t
    ws = torch.full((lib.sa2_distill_workspace_bytes(C.c_int64(70), C.c_int32(5)),), 0x41, dtype=torch.uint8, device="cuda")
    row_loss, total, grad = torch.empty(70, device="cuda"), torch.empty((), device="cuda"), torch.empty_like(z)
    a = DistillArgs(logits=z.data_ptr(), teacher=t.data_ptr(), index=i.data_ptr(), dlogits=grad.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), rows=70,
                    logits_stride=vocab, teacher_stride=5, index_stride=5, dlogits_stride=vocab, vocab=vocab, k=5, index64=1, reduction=forward, temperature=1.5,
                    grad_scale=1.0, stream=torch.cuda.current_stream().cuda_stream)
    a.row_loss = row_loss.data_ptr() if asked != "total" else None
    a.total = total.data_ptr() if asked != "row_loss" else None
    assert lib.sa2_distill_fwd(C.byref(a)) == 0
    a.reduction = backward
    assert lib.sa2_distill_bwd(C.byref(a)) == 0
    leaf = z.requires_grad_()
    loss = lambda reduction: sa.distillation_loss(z.detach(), t, i, temperature=1.5, reduction=reduction)
    assert asked == "total" or torch.equal(row_loss, loss("none"))
    assert asked == "row_loss" or torch.equal(total, loss(("sum", "mean")[forward]))
    want = torch.autograd.grad(sa.distillation_loss(leaf, t, i, temperature=1.5, reduction=("sum", "mean")[backward]), leaf)[0]
    assert torch.equal(grad, want) and (grad[1::3] != 0).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1.0, 20.0, 100.0])
@pytest.mark.parametrize("vocab, k", [(256, 256), (1024, 1024), (3000, 500), (20000, 1000), (70000, 256)], ids=str)
def test_a_student_next_to_its_teacher(vocab, k, temperature, dtype):
    """k equal logits and nothing else, so that the row's sum is k without a rounding; a teacher that is flat but for a tenth.  What the loss is
    made of cancels to its 10^-4 and less: it is formed in 64 bits (10^-13 for a few hundred roundings of numbers below ten) and rounded once."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    z = torch.full((20, vocab), float("-inf"), device="cuda", dtype=dtype)
    z[:, :k] = 0.0
    t = 0.1 * torch.randn(20, k, generator=gen, device="cuda")
    i = torch.stack([torch.randperm(k, generator=gen, device="cuda") for _ in range(20)])
    want = _oracle(z, t, i, temperature)[0]
    bound = want.abs() * 2 * U + temperature ** 2 * 1e-13
    got = sa.distillation_loss(z, t, i, temperature=temperature, reduction="none")
    assert ((got.double() - want).abs() <= bound).all()
    for total in (sa.distillation_loss(z, t, i, temperature=temperature), sa.distillation_loss_and_grad(z, t, i, temperature=temperature)[0]):
        assert (total.double() - want.mean()).abs() <= bound.mean() + want.mean().abs() * 2 * U


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 5001])
@pytest.mark.parametrize("below", [50.0, 104.0, 300.0, 740.0])
def test_ruled_out_tokens_of_little_probability(below, vocab, dtype):
    """An entry `below` nats under the best has a probability of exp(-below), 0 in fp32 from 104 on; the student's -inf there makes the loss inf."""
    z, t, i = _inputs(4, vocab, 5, dtype)
    t[:, 0], t[:, 1:] = 0.0, -below
    z[1, i[1, 3]] = float("-inf")
    loss = sa.distillation_loss(z, t, i, reduction="none")
    assert torch.equal(loss == float("inf"), torch.tensor([False, True, False, False], device="cuda")) and not loss.isnan().any()
    leaf = z.requires_grad_()
    grad = torch.autograd.grad(sa.distillation_loss(leaf, t, i), leaf)[0]
    total, both = sa.distillation_loss_and_grad(z.detach(), t, i)
    assert total == float("inf") and grad.isfinite().all() and both.isfinite().all()
    keep = [0, 2, 3]
    _check(z.detach()[keep], t[keep], i[keep], 1.0, "none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [301, 2047, 5001, 20001, 40003, 70001])
def test_every_place_of_a_row_counts_once(vocab, dtype):
    """A row that one logit dominates, at each place where the reading of a row begins, ends or changes its step, in rows that begin at every distance from a
    16-byte boundary: left out or taken twice, it would change loss and gradient by a third."""
    size, threads = torch.finfo(dtype).bits // 8, (32, 128, 256, 512)
    places = []
    for r in range(8):                                   # (an odd vocabulary: eight rows have all distances)
        head = (-r * vocab * size % 16) // size
        pieces = (vocab - head) // 8
        ends = {0, head - 1, head, head + 7, head + 8, head + 8 * pieces - 9, head + 8 * pieces - 8, head + 8 * pieces - 1, head + 8 * pieces, vocab - 1, vocab // 2}
        ends |= {head + 8 * g * v + d for g in threads for v in (1, 2, 4, 8) for d in (-1, 0) if g * v < pieces}
        ends |= {head + 8 * (pieces - 1 - g * v) + d for g in threads for v in (1, 2, 4, 8) for d in (7, 8) if g * v < pieces}
        places.append(sorted(p for p in ends if 0 <= p < vocab))
    count = max(map(len, places))
    where = torch.tensor([places[r % 8][(r // 8) % len(places[r % 8])] for r in range(8 * count)], device="cuda")
    z, t, i = _inputs(8 * count, vocab, 4, dtype, spread=0.5)
    z.scatter_(1, where[:, None], torch.full_like(z[:, :1], math.log(vocab) + 1))
    i[::2, 0] = where[::2]
    i[:, 1:] = torch.where(i[:, 1:] == i[:, :1], torch.full_like(i[:, 1:], -1), i[:, 1:])
    _check(z, t, i)
