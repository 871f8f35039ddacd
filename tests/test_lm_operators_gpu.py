"""The operators around the attention layers as the language model uses them: tokens in, rotated queries and keys, a teacher's logits or a
sampled token at the end."""
import pytest
import torch
import torch.nn.functional as F

import simplicial_attention_b200 as sa
from simplicial_attention_b200.transformer import Attention, TwoSimplicialLM, training_step


def _lm(rotary=False, **kw):
    return TwoSimplicialLM(num_tokens=256, dim=128, depth=4, max_seq_len=64, dim_head=32, heads=4, two_simplicial_attn_every=2,
                           transformer_kwargs=dict(key_value_heads=2, two_simplicial_attn_kwargs=dict(w1=16, w2=4), attn_kwargs=dict(qk_norm_rotary=rotary)), **kw)


def _teacher(model, tokens, k):
    with torch.no_grad():
        top = model(tokens).float().topk(k, dim=-1)
    return top.values, top.indices


def test_rotated_layer_without_a_gpu():
    torch.manual_seed(1)
    layer = Attention(dim=64, dim_head=16, heads=4, key_value_heads=2, qk_norm_rotary=True)
    assert {"q_norm.weight", "k_norm.weight"} <= set(layer.state_dict()) and "freqs" not in layer.state_dict()
    x = torch.randn(2, 9, 64)
    full = layer(x)
    out, cache = layer(x[:, :6], return_cache=True)
    steps = [out]
    for t in range(6, 9):
        o, cache = layer(x[:, t:t + 1], cache=cache, return_cache=True)
        steps.append(o)
    assert torch.allclose(torch.cat(steps, dim=1), full, atol=1e-5)
    plain = Attention(dim=64, dim_head=16, heads=4, key_value_heads=2)
    plain.load_state_dict({k: v for k, v in layer.state_dict().items() if "_norm" not in k})
    assert not torch.allclose(plain(x), full, atol=1e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_embeddings_are_the_modules(dtype):
    torch.manual_seed(0)
    model = _lm().cuda().to(dtype)
    x = torch.randint(0, 256, (3, 40), device="cuda")
    want = model.token_emb(x) + model.pos_emb(torch.arange(7, 47, device="cuda"))
    assert torch.equal(model._embed(x, 7), want)
    model.token_emb.register_forward_hook(lambda m, a, out: out * 0)         # a hook is seen
    assert torch.equal(model._embed(x, 7), model.pos_emb(torch.arange(7, 47, device="cuda")).expand(3, 40, 128))


@pytest.mark.gpu
def test_embedding_gradients_in_a_step():
    """fp32 sums of the same terms in another order: at most 120 of them a row, each off by 2^-24."""
    torch.manual_seed(0)
    model = _lm(embed_scale=2.0).cuda()
    x = torch.randint(0, 9, (3, 41), device="cuda")
    grads = []
    for hooked in (False, True):
        model.zero_grad()
        handle = model.pos_emb.register_forward_hook(lambda m, a, out: None) if hooked else None
        model(x, return_loss=True).backward()
        if handle is not None:
            handle.remove()
        grads.append((model.token_emb.weight.grad, model.pos_emb.weight.grad))
    for a, b in zip(*grads):
        assert (a - b).abs().max() <= 120 * 2.0 ** -24 * b.abs().max() * 10


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [False, True], ids=["f32", "autocast"])
def test_rotated_model_cached_and_trained(autocast):
    torch.manual_seed(2)
    model = _lm(rotary=True).cuda()
    tokens = torch.randint(0, 256, (2, 40), device="cuda")
    with torch.no_grad():
        full = model(tokens)
        logits, cache = model(tokens[:, :21], return_cache=True)
        got = [logits]
        for t in range(21, 40):
            step, cache = model(tokens[:, t:t + 1], cache=cache, return_cache=True)
            got.append(step)
    assert (torch.cat(got, dim=1) - full).abs().max() <= 1e-3 * full.abs().max()
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        loss = model(tokens, return_loss=True)
    loss.backward()
    layer = model.transformer.layers[0][0]
    for p in (layer.q_norm.weight, layer.k_norm.weight, layer.to_q.weight, layer.to_kv.weight):
        assert p.grad.isfinite().all() and (p.grad != 0).any()


@pytest.mark.gpu
def test_rotated_layer_against_the_plain_form():
    torch.manual_seed(3)
    layer = Attention(dim=64, dim_head=64, heads=4, key_value_heads=2, qk_norm_rotary=True)
    x = torch.randn(2, 30, 64)
    want = layer(x)
    got = layer.cuda()(x.cuda()).cpu()
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.gpu
def test_a_step_against_a_teacher():
    """tokens -> embeddings -> rotated layers -> the teacher's loss, through autograd and as one call."""
    torch.manual_seed(4)
    teacher, model = _lm().cuda(), _lm(rotary=True).cuda()
    tokens = torch.randint(0, 256, (4, 33), device="cuda")
    values, index = _teacher(teacher, tokens[:, :-1], 16)
    index[1, 20:] = -1                                   # padding
    loss = model(tokens, return_loss=True, teacher_logits=values, teacher_index=index, temperature=2.0)
    loss.backward()
    grads = [p.grad.clone() for p in model.parameters()]
    # the same from torch's operators
    model.zero_grad()
    logits = model(tokens[:, :-1]) / 2.0
    p = torch.softmax(values / 2.0, -1)
    log_q = torch.log_softmax(logits, -1).gather(-1, index.clamp_min(0))
    rows = (index[..., 0] >= 0).float()
    want = 4.0 * ((p * (p.log() - log_q)).sum(-1) * rows).sum() / rows.sum()
    want.backward()
    assert (loss - want).abs() <= 1e-5 * want.abs()
    for a, p in zip(grads, model.parameters()):
        assert (a - p.grad).abs().max() <= 1e-4 * p.grad.abs().max() + 1e-7
    model.zero_grad()
    before = [p.detach().clone() for p in model.parameters()]
    opt = torch.optim.SGD(model.parameters(), lr=1.0)
    again = training_step(model, opt, tokens, max_grad_norm=1e9, teacher_logits=values, teacher_index=index, temperature=2.0)
    assert (again - loss).abs() <= 1e-5 * loss.abs()
    for b, g, p in zip(before, grads, model.parameters()):
        assert ((b - p) - g).abs().max() <= 1e-4 * g.abs().max() + 1e-6
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert training_step(model, opt, tokens, teacher_logits=values, teacher_index=index).isfinite()


@pytest.mark.gpu
def test_sampling_with_filters():
    torch.manual_seed(5)
    model = _lm(rotary=True).cuda().eval()
    prompt = torch.randint(0, 256, (3, 10), device="cuda")
    gen = lambda: torch.Generator(device="cuda").manual_seed(11)
    a = model.sample(prompt, 30, temperature=0.9, top_p=0.95, min_p=0.01, generator=gen())
    b = model.sample(prompt, 30, temperature=0.9, top_p=0.95, min_p=0.01, generator=gen())
    assert a.shape == (3, 20) and torch.equal(a, b) and (a >= 0).all() and (a < 256).all()
    c = model.sample(prompt, 30, temperature=0.9, top_k=256, generator=gen())
    assert c.shape == (3, 20)
    # one token kept: the largest logit of every step, by hand
    for use_cache in (True, False):
        out, cache = prompt, None
        with torch.no_grad():
            for _ in range(20):
                if use_cache:
                    logits, cache = model(out if cache is None else out[:, -1:], cache=cache, return_cache=True)
                else:
                    logits = model(out)
                out = torch.cat((out, logits[:, -1].argmax(-1, keepdim=True)), dim=-1)
        assert torch.equal(model.sample(prompt, 30, top_k=1, use_cache=use_cache), out[:, 10:])
        assert torch.equal(model.sample(prompt, 30, temperature=0.0, top_p=0.9, use_cache=use_cache), out[:, 10:])
    # step by step: what the first token is drawn from
    with torch.no_grad():
        logits = model(prompt)[:, -1]
    first = sa.sample_tokens(logits, torch.rand(3, device="cuda", generator=gen()), temperature=0.9, top_p=0.95, min_p=0.01)
    assert torch.equal(a[:, 0], first)


@pytest.mark.gpu
def test_a_generation_step_as_a_graph():
    """Embedding, norm and rotation, sampling: captured once, replayed on new inputs."""
    torch.manual_seed(6)
    b, vocab, dim, heads, d = 4, 1000, 128, 2, 64
    table, head = torch.randn(vocab, dim, device="cuda").bfloat16(), torch.randn(vocab, heads * d, device="cuda").bfloat16()
    gain, freqs = torch.ones(d, device="cuda"), sa.rotary_frequencies(d, device="cuda")
    tokens, places, u = torch.randint(0, vocab, (b, 1), device="cuda"), torch.randint(0, 500, (b, 1), device="cuda"), torch.rand(b, device="cuda")

    def step():
        x = sa.token_embedding(tokens, table, scale=dim ** 0.5).view(b, 1, heads, d)
        q, k = sa.qk_norm_rotary(x, x, gain, gain, freqs, positions=places)
        return sa.sample_tokens(F.linear((q + k).view(b, -1), head), u, top_k=50, top_p=0.9)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        tokens.random_(0, vocab)
        places.random_(0, 10 ** 6)
        u.uniform_()
        graph.replay()
        assert torch.equal(out.clone(), step())


@pytest.mark.gpu
def test_threads_at_once():
    """Calls with little and with much shared memory from several threads, each on its stream: the results of calls one by one."""
    import threading

    gen = torch.Generator(device="cuda").manual_seed(3)
    cases = []
    for vocab, k in ((3000, 4), (3000, 1024), (9000, 300), (40000, 32)):
        z = torch.randn(40, vocab, generator=gen, device="cuda")
        cases.append((z, torch.randn(40, k, generator=gen, device="cuda"), torch.randint(vocab, (40, k), generator=gen, device="cuda"),
                      torch.rand(40, generator=gen, device="cuda")))

    def run(z, t, i, u):
        return (*sa.distillation_loss_and_grad(z, t, i), sa.sample_tokens(z, u, top_k=40, top_p=0.9))

    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(case, expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got = run(*case)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                        wrong.append("results differ")
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(c, w)) for c, w in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_hooks_and_other_modules_of_the_norms(device):
    torch.manual_seed(8)
    layer = Attention(dim=64, dim_head=32, heads=4, key_value_heads=2, qk_norm_rotary=True).to(device)
    x = torch.randn(2, 9, 64, device=device)
    want = layer(x)
    seen = []
    for m in (layer.q_norm, layer.k_norm):
        m.register_forward_hook(lambda m, a, out: seen.append(m))
        m.register_full_backward_hook(lambda m, a, g: seen.append(m))
    got = layer(x)
    assert seen == [layer.q_norm, layer.k_norm] and (got - want).abs().max() <= 1e-4 * want.abs().max()
    got.sum().backward()
    assert len(seen) == 4
    # a module's result is what is turned
    layer.k_norm.register_forward_hook(lambda m, a, out: out * 0)
    assert (layer(x)[:, 0] - want[:, 0]).abs().max() <= 1e-4 * want.abs().max() and not torch.allclose(layer(x)[:, 1:], want[:, 1:], atol=1e-3)
    other = Attention(dim=64, dim_head=32, heads=4, key_value_heads=2, qk_norm_rotary=True).to(device)
    other.load_state_dict(layer.state_dict())
    other.k_norm.eps = 10.0
    assert not torch.allclose(other(x)[:, 1:], want[:, 1:], atol=1e-3)
    other.q_norm, other.k_norm = torch.nn.Identity(), torch.nn.Identity()
    q, k = (f(other.prenorm(x)).view(2, 9, -1, 32) for f in (other.to_q, lambda y: other.to_kv(y).chunk(2, -1)[0]))
    got = other._norm_rotate(q, k, 5)
    for a, b in zip(got, (q, k)):
        assert torch.allclose(a.norm(dim=-1), b.norm(dim=-1), rtol=1e-5) and not torch.allclose(a, b, atol=1e-2)
