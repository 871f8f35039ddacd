"""Embedding lookup and its gradients against 64 bits.

Tolerances count roundings: a result is rounded to its type (half a step), the scale and a product to fp32, and a sum of m
terms in fp32 in any order is off by at most m 2^-24 of the sum of their magnitudes."""
import pytest
import torch

import simplicial_attention_b200 as sa
from simplicial_attention_b200 import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _half_step(t):
    return torch.finfo(t.dtype).eps / 2


def _case(shape, vocab, dim, dtype, positions=0, seed=0, tokens=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    weight = torch.randn(vocab, dim, generator=gen, device="cuda").to(dtype).requires_grad_()
    pos = torch.randn(positions, dim, generator=gen, device="cuda").to(dtype).requires_grad_() if positions else None
    if tokens is None:
        tokens = (vocab ** torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64)).long().clamp_(1, vocab) - 1
    dout = torch.randn(*tokens.shape, dim, generator=gen, device="cuda").to(dtype)
    return tokens, weight, pos, dout


def _check(tokens, weight, pos, dout, scale=1.0, start=0, padding_idx=None):
    vocab, dim = weight.shape
    out = sa.token_embedding(tokens, weight, pos, scale=scale, start=start, padding_idx=padding_idx)
    leaves = [weight] if pos is None else [weight, pos]
    grads = torch.autograd.grad(out, leaves, dout)
    flat = tokens.long().flatten()
    there = (flat >= 0) & (flat < vocab)
    n = tokens.shape[-1]
    scaled = weight.detach().double()[flat.clamp(0, vocab - 1)] * scale
    want = scaled.view(*tokens.shape, dim)
    if pos is not None:
        want = want + pos.detach().double()[start:start + n]
    bound = want.abs() * _half_step(out) * (1 + 2 ** -7) + (2 * U * scaled.abs()).view_as(want)
    ok = there.view(tokens.shape)
    assert ((out.double() - want).abs() <= bound)[ok].all()
    assert out[~ok].isnan().all()

    d = dout.double().flatten(0, -2)
    has = there if padding_idx is None else there & (flat != padding_idx)
    sums, sizes, count = (torch.zeros(vocab, dim, dtype=torch.float64, device="cuda") for _ in range(3))
    sums.index_add_(0, flat[has], d[has])
    sizes.index_add_(0, flat[has], d[has].abs())
    count.index_add_(0, flat[has], torch.ones_like(d[has]))
    bound = (count + 3) * U * sizes * abs(scale) + (sums * scale).abs() * _half_step(weight) * (1 + 2 ** -7)
    assert ((grads[0].double() - sums * scale).abs() <= bound).all()
    assert (grads[0][count[:, 0] == 0] == 0).all()
    if pos is not None:
        rows = d.view(-1, n, dim)
        bound = (rows.shape[0] + 3) * U * rows.abs().sum(0) + rows.sum(0).abs() * _half_step(pos) * (1 + 2 ** -7)
        assert ((grads[1][start:start + n].double() - rows.sum(0)).abs() <= bound).all()
        assert (grads[1][:start] == 0).all() and (grads[1][start + n:] == 0).all()
    return out, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape, vocab, dim, positions, start", [
    ((1, 1), 1, 8, 0, 0),               # one token of one
    ((1, 1), 5, 1, 3, 2),               # a single channel, the last position
    ((2, 17), 3, 64, 20, 3),            # every token many times
    ((1, 31), 40, 72, 0, 0), ((1, 32), 40, 72, 0, 0), ((1, 33), 40, 72, 33, 0),         # around a stretch
    ((3, 1025), 255, 260, 1030, 5),     # four channels behind the last eight: rows of any alignment in bf16
    ((2, 700), 511, 65, 700, 0),        # odd rows
    ((2, 700), 512, 2056, 0, 0),        # the first size with a tenth bit of keys, more than 256 lanes
    ((5, 4096), 256, 96, 0, 0),         # sixteen CTAs sort
    ((1, 3000), 70001, 40, 0, 0),
    ((1, 2000), 300001, 8, 0, 0),       # three passes
], ids=str)
def test_lookup_and_gradients(shape, vocab, dim, positions, start, dtype):
    _check(*_case(shape, vocab, dim, dtype, positions), scale=1.0 if positions else dim ** 0.5, start=start)


@pytest.mark.parametrize("dim", [64, 33])
def test_one_token_everywhere(dim):
    tokens = torch.full((4, 3001), 7, device="cuda")
    _check(*_case(None, 9, dim, torch.float32, tokens=tokens))


@pytest.mark.parametrize("dim", [128, 5])
def test_all_tokens_differ_and_runs_of_a_stretch(dim):
    _check(*_case(None, 4096, dim, torch.bfloat16, tokens=torch.randperm(4096, device="cuda").view(4, 1024)))
    _check(*_case(None, 64, dim, torch.bfloat16, tokens=torch.arange(64, device="cuda").repeat_interleave(32).view(2, 1024)))


@pytest.mark.parametrize("dim", [64, 7])
def test_tokens_outside_and_padding(dim):
    tokens, weight, pos, dout = _case((3, 400), 50, dim, torch.float32, 400)
    tokens[0, :70] = -1
    tokens[1, 5:80] = 50
    tokens[2, 9] = 2 ** 40
    tokens[2, 30:200] = 3
    # places outside carry NaN from above too: nobody reads them for the table
    dout[0, :70] = 1.0
    _check(tokens, weight, pos, dout, padding_idx=3)
    tokens.fill_(-100)
    _, grads = _check(tokens, weight, pos, dout)
    assert (grads[0] == 0).all()


def test_int32_strided_and_one_dimension():
    tokens, weight, pos, dout = _case((6, 50), 30, 40, torch.bfloat16, 50)
    a = sa.token_embedding(tokens, weight, pos, scale=0.5)
    assert torch.equal(a, sa.token_embedding(tokens.int(), weight, pos, scale=0.5))
    assert torch.equal(a, sa.token_embedding(tokens.t().contiguous().t(), weight, pos, scale=0.5))
    assert torch.equal(a[2], sa.token_embedding(tokens[2], weight, pos, scale=0.5))
    assert torch.equal(a[2, 0], sa.token_embedding(tokens[2, 0], weight, pos, scale=0.5))
    # a table that begins and ends anywhere, and every other row of one
    wide = torch.randn(61, 41, device="cuda").bfloat16()
    assert torch.equal(sa.token_embedding(tokens, wide[1::2, 1:]), wide[1::2, 1:][tokens])


def test_empty():
    weight = torch.randn(5, 8, device="cuda", requires_grad=True)
    pos = torch.randn(4, 8, device="cuda", requires_grad=True)
    out = sa.token_embedding(torch.zeros(3, 0, dtype=torch.long, device="cuda"), weight, pos)
    assert out.shape == (3, 0, 8)
    for g in torch.autograd.grad(out, [weight, pos], torch.zeros_like(out)):
        assert (g == 0).all()


@pytest.mark.parametrize("frozen", ["weight", "pos"])
def test_one_table_frozen(frozen):
    tokens, weight, pos, dout = _case((4, 100), 30, 64, torch.float32, 120)
    _, both = _check(tokens, weight, pos, dout, start=7)
    (weight if frozen == "weight" else pos).requires_grad_(False)
    kept = pos if frozen == "weight" else weight
    got = torch.autograd.grad(sa.token_embedding(tokens, weight, pos, start=7), kept, dout)[0]
    assert torch.equal(got, both[1 if frozen == "weight" else 0])


def test_same_bits_from_run_to_run_and_on_another_stream():
    tokens, weight, pos, dout = _case((16, 1024), 256, 512, torch.float32, 1024)
    _, first = _check(tokens, weight, pos, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(sa.token_embedding(tokens, weight, pos), [weight, pos], dout)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_backward_of_the_backward():
    tokens, weight, pos, dout = _case((2, 30), 11, 16, torch.float32, 40)
    dout.requires_grad_()
    for f in (lambda: sa.token_embedding(tokens, weight, pos, scale=2.0, start=4),
              lambda: 2.0 * torch.nn.functional.embedding(tokens, weight) + pos[4:34]):
        grads = torch.autograd.grad(f(), [weight, pos], dout, create_graph=True)
        second = torch.autograd.grad(sum(g.square().sum() for g in grads), dout)[0]
        if "want" in locals():
            # sums of at most 60 terms, twice: 2^-24 of each
            assert (second - want).abs().max() <= 200 * U * want.abs().max()
        want = second


def test_backward_of_the_backward_with_tokens_outside():
    tokens, weight, _, dout = _case((2, 30), 11, 16, torch.float32)
    tokens[0, :9] = -1
    tokens[1, 3] = 11
    tokens[1, 5:8] = 4
    dout.requires_grad_()
    out = sa.token_embedding(tokens, weight, padding_idx=4)
    grad = torch.autograd.grad(out, weight, dout, create_graph=True)[0]
    second = torch.autograd.grad(grad.square().sum(), dout)[0]
    counts = (tokens >= 0) & (tokens < 11) & (tokens != 4)
    assert (second[~counts] == 0).all() and (second[counts] != 0).any()
    plain = torch.autograd.grad(sa.token_embedding(tokens, weight, padding_idx=4), weight, dout)[0]
    assert (grad - plain).abs().max() <= 60 * U * plain.abs().max() * 4


def test_padding_from_the_end():
    tokens, weight, _, dout = _case((2, 30), 11, 16, torch.float32)
    tokens[0, :5] = 10
    got = [torch.autograd.grad(sa.token_embedding(tokens, weight, padding_idx=x), weight, dout)[0] for x in (10, -1)]
    assert torch.equal(*got) and (got[0][10] == 0).all()


def test_captured():
    tokens, weight, pos, dout = _case((4, 600), 100, 64, torch.bfloat16, 600)
    weight, pos = weight.detach(), pos.detach()
    args = [weight.clone().requires_grad_(), pos.clone().requires_grad_()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(sa.token_embedding(tokens, *args), args, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sa.token_embedding(tokens, *args)
        grads = torch.autograd.grad(out, args, dout)
    for seed in (1, 2):
        other = _case((4, 600), 100, 64, torch.bfloat16, 600, seed=seed)
        tokens.copy_(other[0])
        dout.copy_(other[3])
        graph.replay()
        want_out, want = _check(tokens, weight.requires_grad_(), pos.requires_grad_(), dout)
        assert torch.equal(out, want_out) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_wrong_c_calls_are_status_codes():
    import ctypes as C
    lib = _lib.lib()
    assert lib.sa2_embed_fwd(None) == 1 and lib.sa2_embed_bwd(None) == 1
    lib.sa2_embed_workspace_bytes.restype = C.c_size_t
    assert lib.sa2_embed_workspace_bytes(C.c_int64(0), C.c_int32(8)) == 0
    assert lib.sa2_embed_workspace_bytes(C.c_int64(100), C.c_int32(8)) >= 4 * 400 + 4 * 2 * 8 * 4


def test_positions_behind_the_table_are_refused():
    tokens, weight, pos, _ = _case((2, 30), 11, 16, torch.float32, 40)
    for start in (11, 2 ** 63 - 1, 2 ** 63 - 30):
        with pytest.raises(ValueError, match="positions"):
            sa.token_embedding(tokens, weight, pos, start=start)
    assert sa.token_embedding(tokens, weight, pos, start=10).shape == (2, 30, 16)


def _c_backward(tokens, vocab, dim, dtype, positions=0):
    """The C entry's gradients in memory that held NaN, and a call that repeats it."""
    import ctypes as C

    from test_operator_refusals import EmbedArgs
    lib = _lib.lib()
    lib.sa2_embed_workspace_bytes.restype = C.c_size_t
    dout = torch.randn(*tokens.shape, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    dweight = torch.full((vocab, dim), float("nan"), device="cuda", dtype=dtype)
    dpositions = torch.full((positions, dim), float("nan"), device="cuda", dtype=dtype)
    ws = torch.empty(lib.sa2_embed_workspace_bytes(C.c_int64(tokens.numel()), C.c_int32(dim)), dtype=torch.uint8, device="cuda")
    a = EmbedArgs(tokens=tokens.data_ptr(), dout=dout.data_ptr(), dweight=dweight.data_ptr(), dpositions=dpositions.data_ptr() if positions else None, workspace=ws.data_ptr(),
                  workspace_bytes=ws.numel(), rows=tokens.numel(), vocab=vocab, n=tokens.shape[-1], dim=dim, position_rows=positions, tokens64=1, padding=-1, scale=1.0,
                  dtype=_lib.SA2_F32 if dtype == torch.float32 else _lib.SA2_BF16, stream=torch.cuda.current_stream().cuda_stream)

    def call():
        assert lib.sa2_embed_bwd(C.byref(a)) == 0

    call()
    return call, dout, dweight, dpositions, ws


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 33, 700, 3000])
@pytest.mark.parametrize("vocab, dim", [(1, 4096), (2, 70000), (65, 8200), (333, 4096), (5003, 4096), (8192, 1000), (8191, 2049), (40009, 1031), (300007, 65)], ids=str)
def test_zeros_of_tokens_that_are_not_there(vocab, dim, rows, dtype):
    """Wide and narrow tables around the sizes at which more CTAs share the zeros: each row of the gradient is written, by one of them."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    tokens = torch.randint(vocab, (1, rows), generator=gen, device="cuda")
    tokens[0, 0] = vocab - 1
    for positions in (0, rows + 3):
        _, dout, dweight, dpositions, _ = _c_backward(tokens, vocab, dim, dtype, positions)
        count = torch.bincount(tokens[0], minlength=vocab)
        assert (dweight[count == 0] == 0).all()
        once = (count == 1).nonzero()[:, 0]
        place = torch.empty(vocab, dtype=torch.long, device="cuda").scatter_(0, tokens[0], torch.arange(rows, device="cuda"))
        assert torch.equal(dweight[once], dout[0, place[once]]) and not dweight.isnan().any()
        if positions:
            assert torch.equal(dpositions[:rows], dout[0]) and (dpositions[rows:] == 0).all()


@pytest.mark.parametrize("vocab", [8192, 128000])
def test_few_tokens_of_a_wide_table_cost_little_more_than_its_zeros(vocab):
    """A step with a handful of tokens is bound by the zeros of the dense gradient, whatever the table's shape: with CTAs counted by the vocabulary alone,
    one token of 8192 took seven times the time of a fill."""
    call, _, dweight, _, ws = _c_backward(torch.tensor([[5]], device="cuda"), vocab, 4096, torch.float32)

    def best(f):
        times = []
        for _ in range(10):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            f()
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert best(call) <= 3 * best(dweight.zero_)
