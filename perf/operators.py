"""The parts of a language model around its attention layers, as cases that can be timed and whose outputs can be compared.

Four operators of a decoder such as ``TwoSimplicialLM``, from the tokens to what the logits are used for:

  embed     rows of the embedding table times a scale, plus the learned positions; in training the dense gradients of both tables;
  rotary    RMSNorm of every query and key head and the rotation by position behind it; in training with the gradients of
            queries, keys and both gains;
  distill   T^2 KL(teacher || student) against the teacher's K largest logits of a position, with the gradient of the student's
            logits, through autograd ("form": "autograd") or both from one call ("form": "both");
  sample    a token for each row of logits: temperature, top-k, top-p and min-p, drawn with a given uniform number, and the logarithm
            of the probability that it had.

``run`` has each in plain torch (``own`` false) and as the package's call (``own`` true).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"bf16": 2, "f32": 4}


def _embed(b, n, vocab, dim, dtype, positions, train):
    return {"kind": "embed", "b": b, "n": n, "vocab": vocab, "dim": dim, "dtype": dtype, "positions": positions, "train": train}


def _rotary(b, n, hq, hk, d, rotated, dtype, start, interleaved, train):
    return {"kind": "rotary", "b": b, "n": n, "hq": hq, "hk": hk, "d": d, "rotated": rotated, "dtype": dtype, "start": start,
            "interleaved": interleaved, "train": train}


def _distill(rows, vocab, k, dtype, temperature, form):
    return {"kind": "distill", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype, "temperature": temperature, "form": form}


def _sample(rows, vocab, dtype, temperature, top_k, top_p, min_p):
    return {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "top_k": top_k, "top_p": top_p,
            "min_p": min_p}


def listed():
    return [
        # a generated token of 32 sequences enters the model: all latency
        dict(_embed(32, 1, 32000, 1024, "bf16", True, False), name="embed_step"),
        # the byte model's training batch: few table rows, each with many tokens
        dict(_embed(16, 1024, 256, 512, "f32", True, True), name="embed_train_bytes"),
        # a large vocabulary of odd size, scaled embeddings: most of the dense gradient is zeros
        dict(_embed(4, 4096, 50001, 2048, "bf16", False, True), name="embed_train_large"),
        # a generated token of 32 sequences of different lengths in a standard layer: all latency
        dict(_rotary(32, 1, 8, 4, 64, 64, "bf16", 700, False, False), name="rotary_step"),
        # a standard layer of the 8-layer decoder, forward and backward
        dict(_rotary(16, 1024, 8, 4, 64, 64, "bf16", 0, False, True), name="rotary_train"),
        # a stretch of a long prompt, odd length, half of the channels rotated, neighbouring channels paired
        dict(_rotary(2, 5001, 16, 4, 128, 64, "f32", 100000, True, False), name="rotary_prefill"),
        # the byte model's training batch against a teacher's eight largest logits
        dict(_distill(16384, 256, 8, "bf16", 1.0, "autograd"), name="distill_bytes"),
        # fp32 logits of a usual vocabulary, odd number of rows
        dict(_distill(4095, 32000, 32, "f32", 2.0, "autograd"), name="distill_train"),
        # a step over a large vocabulary, loss and gradient from one call: the largest
        dict(_distill(4096, 128000, 64, "bf16", 2.0, "both"), name="distill_step"),
        # one sequence of the byte model, a tenth of the vocabulary kept: the smallest call, all latency
        dict(_sample(1, 256, "f32", 0.8, 26, 1.0, 0.0), name="sample_b1"),
        # a serving batch with the usual filters
        dict(_sample(64, 32000, "bf16", 0.7, 50, 0.95, 0.0), name="sample_batch"),
        # a large batch and vocabulary, the nucleus and a floor below the best token
        dict(_sample(256, 128000, "f32", 1.0, 0, 0.9, 0.02), name="sample_large"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above: one to 65536 positions, vocabularies of 64 to 131072 tokens, widths of 64 to 4096 channels (one in
    four odd), head dims of 32 to 256, one to 1024 teacher logits, filters on and off."""
    kind = rng.choice(("embed", "rotary", "distill", "sample"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind == "embed":
        dim = _log_int(rng, 64, 4096)
        dim = dim | 1 if rng.random() < 0.25 else max(64, dim // 64 * 64)
        b = _log_int(rng, 1, 64)
        case = _embed(b, _log_int(rng, 1, max(1, 65536 // b)), _log_int(rng, 64, 131072), dim, dtype, rng.random() < 0.5, rng.random() < 0.7)
        while work(case)["bytes"] > 1.5e9:
            case["vocab"], case["n"] = max(64, case["vocab"] * 2 // 3), max(1, case["n"] * 2 // 3)
        return case
    if kind == "rotary":
        hk = rng.choice((1, 2, 3, 4, 8))
        d = rng.choice((32, 64, 64, 128, 128, 256))
        b = _log_int(rng, 1, 32)
        case = _rotary(b, _log_int(rng, 1, max(1, 32768 // b)), hk * rng.choice((1, 2, 3, 4)), hk, d, d // rng.choice((1, 1, 2)), dtype,
                       _log_int(rng, 1, 1000000), rng.random() < 0.4, rng.random() < 0.6)
        while work(case)["bytes"] > 1.5e9:
            case["n"] = max(1, case["n"] * 2 // 3)
        return case
    rows = _log_int(rng, 1, 16384)
    vocab = _log_int(rng, 64, 131072)
    if kind == "distill":
        case = _distill(rows, vocab, min(vocab, _log_int(rng, 1, 1024)), dtype, round(rng.uniform(0.5, 4.0), 2), rng.choice(("autograd", "both")))
        while work(case)["bytes"] > 1.5e9:
            case["rows"] = max(1, case["rows"] * 2 // 3)
        return case
    top_k = rng.choice((0, _log_int(rng, 1, 1000)))
    top_p = rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3)))
    min_p = rng.choice((0.0, round(math.exp(rng.uniform(math.log(0.002), math.log(0.3))), 4)))
    return _sample(max(1, min(rows, 40000000 // vocab)), vocab, dtype, round(rng.uniform(0.3, 1.6), 2), top_k, top_p, min_p)


def work(case):
    """What a pass cannot do without: each input read once, each output written once."""
    kind, size = case["kind"], SIZES[case["dtype"]]
    if kind == "embed":
        tokens, dim = case["b"] * case["n"], case["dim"]
        table = min(tokens, case["vocab"]) * dim
        positions = case["n"] * dim if case["positions"] else 0
        total = 8 * tokens + size * (table + positions + tokens * dim)
        flops = 2 * tokens * dim
        if case["train"]:       # dOut in, both dense gradients out
            total += size * (tokens * dim + case["vocab"] * dim + (_rows_of_positions(case) * dim if case["positions"] else 0))
            flops += 2 * tokens * dim
        return {"bytes": total, "flops": flops}
    if kind == "rotary":
        values = case["b"] * case["n"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": size * values * (4 if case["train"] else 2) + 8 * case["b"] * case["n"], "flops": values * (22 if case["train"] else 8)}
    if kind == "distill":
        values, teacher = case["rows"] * case["vocab"], case["rows"] * case["k"]
        return {"bytes": 2 * size * values + (size + 8) * teacher, "flops": 6 * values + 8 * teacher}
    return {"bytes": case["rows"] * (size * case["vocab"] + 16), "flops": 4 * case["rows"] * case["vocab"]}


def _rows_of_positions(case):
    return case["n"] + 24       # the table is longer than the sequence


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype, times=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(times).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    kind, state = case["kind"], {"case": case}
    if kind == "embed":
        b, n, vocab, dim = (case[k] for k in ("b", "n", "vocab", "dim"))
        # token frequencies of text: the r-th most frequent in proportion to 1 / r, on shuffled ids
        shuffled = torch.randperm(vocab, generator=gen, device="cuda")
        rank = (vocab ** uniform(b, n).double()).long().clamp_(1, vocab) - 1
        state["tokens"] = shuffled[rank]
        state["weight"] = normal(vocab, dim, times=0.02).requires_grad_(case["train"])
        state["positions"] = normal(_rows_of_positions(case), dim, times=0.02).requires_grad_(case["train"]) if case["positions"] else None
        state["scale"] = 1.0 if case["positions"] else math.sqrt(dim)
        state["dout"] = normal(b, n, dim) if case["train"] else None
        return state
    if kind == "rotary":
        b, n, hq, hk, d = (case[k] for k in ("b", "n", "hq", "hk", "d"))
        # queries, keys and values of one fused projection, as a layer has them
        packed = normal(b, n, (hq + 2 * hk) * d)
        state["q"] = packed[..., :hq * d].unflatten(-1, (hq, d)).detach().requires_grad_(case["train"])
        state["k"] = packed[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d)).detach().requires_grad_(case["train"])
        state["gains"] = [(1 + normal(d, dtype=torch.float32, times=0.1)).to(dtype).requires_grad_(case["train"]) for _ in range(2)]
        # every sequence has come to a place of its own
        lengths = (uniform(b, 1) * 300).long() + case["start"]
        state["places"] = lengths + torch.arange(n, device="cuda")
        state["dq"], state["dk"] = (normal(b, n, hq, d), normal(b, n, hk, d)) if case["train"] else (None, None)
        state["inv"] = 10000.0 ** (-torch.arange(0, case["rotated"], 2, device="cuda", dtype=torch.float64) / case["rotated"])
        if own:
            from simplicial_attention_b200 import rotary_frequencies
            state["freqs"] = rotary_frequencies(case["rotated"], theta=10000.0, device="cuda")
        return state
    rows, vocab = case["rows"], case["vocab"]
    logits = normal(rows, vocab, times=2.0)
    few = min(vocab, 24)
    favoured = (torch.randint(vocab, (rows, 1), generator=gen, device="cuda") + torch.arange(few, device="cuda") * (vocab // few)) % vocab
    logits.scatter_(1, favoured, normal(rows, few, times=3.0) + 7.0)
    if kind == "distill":
        k = case["k"]
        state["logits"] = logits.requires_grad_(case["form"] == "autograd")
        # the teacher's largest logits first, on distinct tokens; it prefers some that the student prefers too
        index = (torch.randint(vocab, (rows, 1), generator=gen, device="cuda") + torch.arange(k, device="cuda") * max(1, vocab // k)) % vocab
        near = min(8, k, few)
        taken = (index[:, near:, None] == favoured[:, None, :near]).any(-1)
        index = torch.cat((favoured[:, :near], torch.where(taken, torch.full_like(index[:, near:], -1), index[:, near:])), dim=1)
        state["teacher"] = (normal(rows, k, dtype=torch.float32).abs_().cumsum(1).mul_(-0.3) + 12.0).to(dtype)
        # padding: one position in sixteen has no teacher
        blank = uniform(rows, 1) < 1 / 16 if rows > 1 else torch.zeros(rows, 1, dtype=torch.bool, device="cuda")
        state["index"] = torch.where(blank, torch.full_like(index, -1), index).contiguous()
        return state
    state["logits"] = logits
    state["uniform"] = uniform(rows)

    def each(value, spread, least, most):       # every request has settings of its own around the case's
        return (value * (1 + spread * (uniform(rows) - 0.5))).clamp_(least, most)

    state["temperature"] = each(case["temperature"], 0.2, 0.1, 2.0)
    state["top_k"] = each(float(case["top_k"]), 0.5, 1, vocab).long() if case["top_k"] else None
    state["top_p"] = each(case["top_p"], 0.1, 0.05, 0.999) if case["top_p"] < 1 else None
    state["min_p"] = each(case["min_p"], 0.5, 0.0, 0.9) if case["min_p"] else None
    return state


def run(state):
    case = state["case"]
    return {"embed": _run_embed, "rotary": _run_rotary, "distill": _run_distill, "sample": _run_sample}[case["kind"]](case, state)


def _run_embed(case, s):
    n, weight, positions = case["n"], s["weight"], s["positions"]
    if own:
        from simplicial_attention_b200 import token_embedding
        out = token_embedding(s["tokens"], weight, positions, scale=s["scale"])
        if not case["train"]:
            return out
        leaves = [weight] if positions is None else [weight, positions]
        return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]
    with torch.no_grad():
        out = weight[s["tokens"]].float() * s["scale"]
        if positions is not None:
            out = out + positions[:n].float()
        out = out.to(weight.dtype)
        if not case["train"]:
            return out
        dout = s["dout"].float()
        dweight = torch.zeros(weight.shape, device=weight.device).index_add_(0, s["tokens"].flatten(), dout.flatten(0, 1)).mul_(s["scale"])
        if positions is None:
            return [out, dweight.to(weight.dtype)]
        dpositions = torch.zeros(positions.shape, device=weight.device)
        dpositions[:n] = dout.sum(0)
        return [out, dweight.to(weight.dtype), dpositions.to(weight.dtype)]


def _pairs(x, rotated, interleaved):
    """The two channels of every rotated pair, and the channels that stay."""
    if interleaved:
        return x[..., 0:rotated:2], x[..., 1:rotated:2], x[..., rotated:]
    return x[..., :rotated // 2], x[..., rotated // 2:rotated], x[..., rotated:]


def _joined(a, b, rest, interleaved):
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _run_rotary(case, s):
    q, k, gains = s["q"], s["k"], s["gains"]
    if own:
        from simplicial_attention_b200 import qk_norm_rotary
        out = qk_norm_rotary(q, k, *gains, s["freqs"], positions=s["places"], eps=1e-6, interleaved=case["interleaved"])
        if not case["train"]:
            return out
        return [out[0].detach(), out[1].detach(), *torch.autograd.grad(out, [q, k, *gains], [s["dq"], s["dk"]])]
    with torch.no_grad():
        rotated, il = case["rotated"], case["interleaved"]
        angle = s["places"].double()[..., None, None] * s["inv"]
        cos, sin = angle.cos().float(), angle.sin().float()
        outs, dins, dgains = [], [], []
        for x, gain, dy in ((q, gains[0], s["dq"]), (k, gains[1], s["dk"])):
            xf, g = x.float(), gain.float()
            rstd = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + 1e-6)
            hat = xf * rstd
            a, b, rest = _pairs(hat * g, rotated, il)
            outs.append(_joined(a * cos - b * sin, b * cos + a * sin, rest, il).to(x.dtype))
            if dy is None:
                continue
            a, b, rest = _pairs(dy.float(), rotated, il)
            back = _joined(a * cos + b * sin, b * cos - a * sin, rest, il)
            dgains.append((back * hat).sum((0, 1, 2)).to(gain.dtype))
            back = back * g
            dins.append((rstd * (back - hat * (back * hat).mean(-1, keepdim=True))).to(x.dtype))
        return [*outs, *dins, *dgains] if case["train"] else tuple(outs)


def _run_distill(case, s):
    logits, teacher, index, t = s["logits"], s["teacher"], s["index"], case["temperature"]
    if own:
        from simplicial_attention_b200 import distillation_loss, distillation_loss_and_grad
        if case["form"] == "both":
            return distillation_loss_and_grad(logits, teacher, index, temperature=t)
        loss = distillation_loss(logits, teacher, index, temperature=t)
        return [loss.detach(), *torch.autograd.grad(loss, [logits])]
    with torch.no_grad():
        z = logits.float() / t
        z = z - z.amax(-1, keepdim=True)
        e = z.exp()
        total = e.sum(-1, keepdim=True)
        there = index >= 0
        place = index.clamp_min(0)
        y = (teacher.float() / t).masked_fill(~there, float("-inf"))
        best = y.amax(-1, keepdim=True)
        y = y - torch.where(best.isinf(), torch.zeros_like(best), best)
        p = y.exp()
        mass = p.sum(-1, keepdim=True)
        p = p / mass.clamp_min(1e-30)
        log_p = y - mass.clamp_min(1e-30).log()
        log_q = z.gather(-1, place) - total.log()
        counted = there.any(-1)
        rows = counted.sum().clamp_min(1).float()
        terms = torch.where(there, p * (log_p - log_q), torch.zeros_like(p)).double()
        loss = (terms.sum() * (t * t) / rows).float()
        grad = e.div_(total).mul_(counted[:, None])
        grad.scatter_add_(-1, place, -p)
        return [loss, grad.mul_(t / rows).to(logits.dtype)]


def _column(value):
    return value if value is None else value[:, None].double()


def _run_sample(case, s):
    if own:
        from simplicial_attention_b200 import sample_tokens
        return sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                             return_logprobs=True)
    z, order = s["logits"].double().sort(dim=-1, descending=True, stable=True)
    x = (z - z[:, :1]) / _column(s["temperature"])
    p = x.exp()
    rank = torch.arange(z.shape[1], device=z.device)
    kept = torch.ones_like(p, dtype=torch.bool)
    if s["top_k"] is not None:
        kept = rank < s["top_k"][:, None]
    if s["top_p"] is not None:
        p_kept = p * kept
        before = p_kept.cumsum(-1) - p_kept
        kept = kept & (before < _column(s["top_p"]) * p_kept.sum(-1, keepdim=True))
    if s["min_p"] is not None:
        kept = kept & (p >= _column(s["min_p"]))
    kept[:, 0] = True
    weight = torch.zeros_like(p).scatter_(1, order, p * kept)
    cdf = weight.cumsum(-1)
    token = (cdf <= _column(s["uniform"]) * cdf[:, -1:]).sum(-1)
    chosen = torch.zeros_like(x).scatter_(1, order, x).gather(1, token[:, None])
    return token, (chosen - cdf[:, -1:].log()).squeeze(1).float()


def exact(case, seed):
    state = prepare(case, seed)
    return {"embed": _exact_embed, "rotary": _exact_rotary, "distill": _exact_distill, "sample": _exact_sample}[case["kind"]](case, state)


def _exact_embed(case, s):
    tokens, weight, positions = s["tokens"], s["weight"].detach().double(), s["positions"]
    out = torch.nn.functional.embedding(tokens, weight) * s["scale"]
    if positions is not None:
        out = out + positions.detach().double()[torch.arange(case["n"], device=out.device)]
    if not case["train"]:
        return out
    # sorted tokens, running sums, differences at the ends of the runs
    flat, dout = tokens.flatten(), s["dout"].double().flatten(0, 1)
    by_token = flat.argsort(stable=True)
    ends = torch.bincount(flat, minlength=case["vocab"]).cumsum(0)
    dweight = torch.empty_like(weight)
    for c in range(0, case["dim"], 256):
        sums = torch.nn.functional.pad(dout[by_token, c:c + 256].cumsum(0), (0, 0, 1, 0))
        run_end = sums[ends]
        dweight[:, c:c + 256] = (run_end - torch.nn.functional.pad(run_end, (0, 0, 1, 0))[:-1]) * s["scale"]
    if positions is None:
        return [out, dweight]
    dpositions = torch.nn.functional.pad(s["dout"].double().sum(0), (0, 0, 0, positions.shape[0] - case["n"]))
    return [out, dweight, dpositions]


def _exact_rotary(case, s):
    rotated, d = case["rotated"], case["d"]
    # the rotation as complex numbers
    phase = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["places"].double()[..., None, None] * s["inv"])

    def forward(x, gain):
        y = x / (x.square().sum(-1, keepdim=True) / d + 1e-6).sqrt() * gain
        turned = y[..., :rotated]
        if case["interleaved"]:
            turned = torch.view_as_real(torch.view_as_complex(turned.unflatten(-1, (-1, 2)).contiguous()) * phase).flatten(-2)
        else:
            turned = torch.complex(*turned.chunk(2, -1)) * phase
            turned = torch.cat((turned.real, turned.imag), dim=-1)
        return torch.cat((turned, y[..., rotated:]), dim=-1)

    ins = [s[k].detach().double().requires_grad_(case["train"]) for k in ("q", "k")]
    gains = [g.detach().double().requires_grad_(case["train"]) for g in s["gains"]]
    outs = [forward(x, g) for x, g in zip(ins, gains)]
    if not case["train"]:
        return tuple(outs)
    grads = torch.autograd.grad(outs, [*ins, *gains], [s["dq"].double(), s["dk"].double()])
    return [*(o.detach() for o in outs), *grads]


def _exact_distill(case, s):
    t, index = case["temperature"], s["index"]
    rows = int((index >= 0).any(-1).sum().clamp_min(1))
    loss, grads = 0.0, []
    for r in range(0, case["rows"], 512):
        logits = s["logits"][r:r + 512].detach().double().requires_grad_()
        place = index[r:r + 512]
        there = place >= 0
        # the teacher as a distribution over the whole vocabulary
        y = s["teacher"][r:r + 512].double() / t
        p = torch.softmax(y.masked_fill(~there, -1e30), -1) * there
        log_q = torch.log_softmax(logits / t, -1).gather(-1, place.clamp_min(0))
        part = (torch.special.xlogy(p, p) - p * log_q).sum() * (t * t / rows)
        grads.append(torch.autograd.grad(part, logits)[0])
        loss = loss + part.detach()
    return [loss, torch.cat(grads)]


def _exact_sample(case, s):
    import numpy as np
    host = {k: None if v is None else v.double().cpu().numpy() for k, v in s.items() if k != "case"}
    tokens, logprobs = np.empty(case["rows"], dtype=np.int64), np.empty(case["rows"])
    for r in range(case["rows"]):
        z = host["logits"][r]
        w = np.exp((z - z.max()) / host["temperature"][r])
        order = np.lexsort((np.arange(z.size), -z))
        count = z.size
        if host["top_k"] is not None:
            count = min(count, int(host["top_k"][r]))
        if host["top_p"] is not None:
            mass = np.cumsum(w[order[:count]])
            count = min(count, int(np.searchsorted(mass, host["top_p"][r] * mass[-1], side="left")) + 1)
        if host["min_p"] is not None:
            count = min(count, max(1, int((w >= host["min_p"][r]).sum())))
        left = np.sort(order[:count])
        mass = np.cumsum(w[left])
        tokens[r] = left[min(int(np.searchsorted(mass, host["uniform"][r] * mass[-1], side="right")), count - 1)]
        logprobs[r] = np.log(w[tokens[r]] / mass[-1])
    return tuple(torch.from_numpy(t).to(s["logits"].device) for t in (tokens, logprobs))
