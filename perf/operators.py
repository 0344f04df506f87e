"""The operators of the language-model training step: sizes, plain forms, exact values.

Three operators are described, each by its mathematics and by the sizes at which a
training or scoring program meets it:

* attention       o = softmax(scale q k^T + mask) v over grouped heads, and its gradients;
* token log probabilities   log p(token), entropy and the most likely alternatives of
                  rows of logits, and the gradient of the first two;
* residual norm   r = x + scale gate * norm(branch), y = norm(r) weight, and its gradients.

`run` computes a case with elementary torch operations in 32 bits, or, where `own` is
true, through `sofa_amd.workloads.kernels`.  `exact` computes it in 64 bits.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the test suite's two-layer decoder: 128 channels in 8 heads, 32 tokens
        dict(name="attention-tiny-step", op="attention", batch=2, tokens=32, heads=8, kv_heads=2,
             dim=16, causal=True, ragged=False, backward=True),
        # a right-padded batch with an empty sequence, every head with its own keys
        dict(name="attention-padded-step", op="attention", batch=6, tokens=777, heads=16, kv_heads=16,
             dim=64, causal=True, ragged=True, backward=True),
        # the profiled decoder step of the overhead study: 2 sequences of 2048
        dict(name="attention-2k-step", op="attention", batch=2, tokens=2048, heads=32, kv_heads=8,
             dim=128, causal=True, ragged=False, backward=True),
        # the decoder workload's own default: 2 sequences of 4096
        dict(name="attention-4k-step", op="attention", batch=2, tokens=4096, heads=32, kv_heads=8,
             dim=128, causal=True, ragged=False, backward=True),
        # one sequence of the decoder's whole context, evaluated without gradients
        dict(name="attention-8k-forward", op="attention", batch=1, tokens=8192, heads=32, kv_heads=8,
             dim=128, causal=True, ragged=False, backward=False),
        # the distribution behind one sampled token: latency is what counts
        dict(name="logprobs-one-token", op="logprobs", rows=1, vocab=128256, dtype="bf16",
             top=5, masked=False, backward=False),
        # scoring given answers under a vocabulary mask, with alternatives, odd vocabulary
        dict(name="logprobs-score", op="logprobs", rows=500, vocab=50001, dtype="fp32",
             top=20, masked=True, backward=False),
        # the loss of the decoder workload's default step
        dict(name="logprobs-loss-step", op="logprobs", rows=8192, vocab=128256, dtype="bf16",
             top=0, masked=False, backward=True),
        # one token's residual stream: latency is what counts
        dict(name="norm-one-token", op="norm", batch=1, tokens=1, dim=4096, x="fp32", branch="bf16",
             out="bf16", post=False, gate="none", backward=False),
        # the decoder workload's default step under autocast: 32-bit stream, bf16 branch
        dict(name="norm-step", op="norm", batch=2, tokens=4096, dim=4096, x="fp32", branch="bf16",
             out="bf16", post=False, gate="none", backward=True),
        # a block with norms on both sides and a gate for each sequence, odd sizes
        dict(name="norm-gated-step", op="norm", batch=5, tokens=1023, dim=1001, x="bf16", branch="bf16",
             out="bf16", post=True, gate="sequence", backward=True),
        # a layer scale over a whole 32-bit block, channels that do not fill the last vector
        dict(name="norm-scaled-step", op="norm", batch=3, tokens=500, dim=2600, x="fp32", branch="fp32",
             out="fp32", post=False, gate="channel", backward=True),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(("attention", "logprobs", "norm"))
    if op == "attention":
        kv_heads = rng.choice((1, 2, 3, 8))
        heads = kv_heads * rng.choice((1, 2, 4, 5))
        dim = rng.choice((16, 40, 64, 80, 96, 128))
        tokens = _log_uniform(rng, 1, 4096)
        causal = rng.random() < 0.75 or heads * tokens * tokens > 32 * 4096 * 4096
        most = (2 if causal else 1) * 32 * 4096 * 4096 // (heads * tokens * tokens)
        return dict(op=op, batch=_log_uniform(rng, 1, max(1, min(16, most))), tokens=tokens, heads=heads,
                    kv_heads=kv_heads, dim=dim, causal=causal, ragged=rng.random() < 0.4,
                    backward=rng.random() < 0.7)
    if op == "logprobs":
        vocab = _log_uniform(rng, 1000, 160000)
        backward = rng.random() < 0.5
        rows = _log_uniform(rng, 1, min(8192, 8192 * 128256 // vocab))
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        top = 0 if backward else rng.choice((0, 1, 5, 20, 32))
        if top:
            rows = min(rows, 2048)
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=top,
                    masked=rng.random() < 0.3, backward=backward)
    x, branch, out = rng.choice((("fp32", "bf16", "bf16"), ("fp32", "bf16", "fp32"), ("fp32", "fp32", "fp32"),
                                 ("bf16", "bf16", "bf16"), ("fp16", "fp16", "fp16"), ("fp32", "fp16", "fp16")))
    dim = _log_uniform(rng, 64, 8192)
    batch = _log_uniform(rng, 1, 8)
    tokens = _log_uniform(rng, 1, min(4096, 8192 * 4096 // (dim * batch)))
    return dict(op=op, batch=batch, tokens=tokens, dim=dim, x=x, branch=branch, out=out,
                post=rng.random() < 0.5, gate=rng.choice(("none", "channel", "sequence")),
                backward=rng.random() < 0.7)


def _lengths(case):
    """Valid tokens of each sequence: one whole, one empty where there are three or more, the rest spread."""
    n, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t] * n
    return [t if i == 0 else 0 if i == 2 else 1 + (i * 7919 + 263 * t) % t for i in range(n)]


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        x = torch.empty(shape, dtype=torch.float32, device="cuda")
        return x.normal_(mean, std, generator=g).to(dtype)

    state = dict(case=case)
    if case["op"] == "attention":
        b, t, d = case["batch"], case["tokens"], case["dim"]
        # as the projections leave them: (batch, tokens, heads, dim), seen as (batch, heads, tokens, dim)
        for name, h in (("q", case["heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"])):
            state[name] = normal(b, t, h, d, dtype=torch.bfloat16).transpose(1, 2)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        if case["backward"]:
            state["do"] = normal(b, t, case["heads"], d, dtype=torch.bfloat16).transpose(1, 2)
            for name in ("q", "k", "v"):
                state[name].requires_grad_()
    elif case["op"] == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        logits = normal(n, vocab, std=2.5, mean=-1.0)
        if case["masked"]:  # the last twentieth of the vocabulary is not allowed
            logits[:, vocab - vocab // 20:] = -math.inf
        tokens = torch.randint(0, vocab - vocab // 20, (n,), device="cuda", generator=g)
        if n > 4:
            tokens[torch.randint(0, n, (n // 8,), device="cuda", generator=g)] = -100  # prompts, padding
        # a trained model finds its tokens likely
        rows = torch.nonzero(tokens >= 0)[:, 0]
        logits[rows, tokens[rows]] += 6.0
        state["logits"], state["tokens"] = logits.to(TYPES[case["dtype"]]), tokens
        if case["backward"]:
            state["dlogprob"], state["dentropy"] = normal(n), normal(n, std=0.1)
            state["logits"].requires_grad_()
    else:
        b, t, d = case["batch"], case["tokens"], case["dim"]
        loud = 1.0 + 20.0 * (torch.rand(d, device="cuda", generator=g) < 0.01).float()  # a few loud channels
        state["x"] = (normal(b, t, d) * loud).to(TYPES[case["x"]])
        state["branch"] = normal(b, t, d, dtype=TYPES[case["branch"]], std=0.5)
        state["weight"] = normal(d, mean=1.0, std=0.1)
        state["post"] = normal(d, mean=1.0, std=0.1) if case["post"] else None
        state["gate"] = (None if case["gate"] == "none" else normal(d, std=0.5) if case["gate"] == "channel"
                         else normal(b, 1, d, std=0.5, dtype=TYPES[case["branch"]]))
        state["scale"] = 1.0 if case["gate"] == "none" else 0.75
        if case["backward"]:
            state["dr"] = normal(b, t, d, dtype=TYPES[case["x"]])
            state["dy"] = normal(b, t, d, dtype=TYPES[case["out"]])
            for name in ("x", "branch", "weight", "post", "gate"):
                if state[name] is not None:
                    state[name].requires_grad_()
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "logprobs": _own_logprobs, "norm": _own_norm}[op](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "logprobs": _plain_logprobs, "norm": _plain_norm}[op](state)


def _own_attention(s):
    from sofa_amd.workloads import kernels

    o = kernels.attention(s["q"], s["k"], s["v"], lengths=s["lengths"], causal=s["case"]["causal"])
    if not s["case"]["backward"]:
        return (o,)
    return (o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))


def _own_logprobs(s):
    from sofa_amd.workloads import kernels

    out = kernels.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    if s["case"]["backward"]:
        (dx,) = torch.autograd.grad((out.logprob, out.entropy), (s["logits"],), (s["dlogprob"], s["dentropy"]))
        return out.logprob.detach(), out.entropy.detach(), dx
    if s["case"]["top"]:
        return out.logprob, out.entropy, out.top_ids, out.top_logprobs
    return out.logprob, out.entropy


def _own_norm(s):
    from sofa_amd.workloads import kernels

    r, y = kernels.residual_norm(s["x"], s["branch"], s["weight"], post_weight=s["post"], gate=s["gate"],
                                 scale=s["scale"], eps=EPS, out_dtype=TYPES[s["case"]["out"]])
    if not s["case"]["backward"]:
        return r, y
    leaves = [s[n] for n in ("x", "branch", "weight", "post", "gate") if s[n] is not None]
    return (r.detach(), y.detach(), *torch.autograd.grad((r, y), leaves, (s["dr"], s["dy"])))


def _plain_attention(s):
    case = s["case"]
    b, t, d, kv = case["batch"], case["tokens"], case["dim"], case["kv_heads"]
    group = case["heads"] // kv
    scale = 1.0 / math.sqrt(d)
    q = s["q"].float().reshape(b, kv, group * t, d)  # the heads of a group follow each other
    k, v = s["k"].float(), s["v"].float()
    at = torch.arange(t, device=q.device)
    valid = torch.ones(b, t, dtype=torch.bool, device=q.device) if s["lengths"] is None else at[None] < s["lengths"][:, None]
    seen = valid[:, :, None] & valid[:, None, :]
    if case["causal"]:
        seen = seen & (at[None, :, None] >= at[None, None, :])
    seen = seen[:, None, None]  # (batch, 1, 1, tokens, tokens)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(b, kv, group, t, t)
    score.masked_fill_(~seen, -math.inf)
    most = score.amax(-1, keepdim=True)
    score.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = score.sum(-1, keepdim=True)
    p = score.div_(torch.where(total == 0, 1.0, total)).view(b, kv, group * t, t)
    o = torch.matmul(p, v)
    out = o.view(b, kv * group, t, d).to(s["q"].dtype)
    if not case["backward"]:
        return (out,)
    do = s["do"].float().reshape(b, kv, group * t, d)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k).view(b, kv * group, t, d)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    return out, dq.to(s["q"].dtype), dk.to(s["k"].dtype), dv.to(s["v"].dtype)


def _plain_logprobs(s):
    case, tokens = s["case"], s["tokens"]
    x = s["logits"].float()
    e = x - x.amax(-1, keepdim=True)
    total = e.exp().sum(-1, keepdim=True)
    logp = e.sub_(total.log())
    p = logp.exp()
    counted = tokens >= 0
    at = torch.where(counted, tokens, 0)[:, None]
    logprob = torch.where(counted, logp.gather(-1, at)[:, 0], 0.0)
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    if case["backward"]:
        glp = torch.where(counted, s["dlogprob"], 0.0)[:, None]
        gh = s["dentropy"][:, None]
        dx = -glp * p - gh * (plogp + p * entropy[:, None])
        dx.scatter_add_(-1, at, glp)
        return logprob, entropy, dx.to(s["logits"].dtype)
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]]
        return logprob, entropy, ids, logp.gather(-1, ids)
    return logprob, entropy


def _plain_norm(s):
    case, d = s["case"], s["case"]["dim"]
    x, branch, weight = s["x"].float(), s["branch"].float(), s["weight"].float()
    h = branch
    if s["post"] is not None:
        rstd_h = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        unit_h = h * rstd_h
        h = unit_h * s["post"].float()
    gate = s["scale"] if s["gate"] is None else s["gate"].float() * s["scale"]
    r = x + h * gate
    rstd = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    unit = r * rstd
    y = unit * weight
    first = r.to(s["x"].dtype), y.to(TYPES[case["out"]])
    if not case["backward"]:
        return first
    dy = s["dy"].float()
    dunit = dy * weight
    dr = s["dr"].float() + rstd * (dunit - unit * (dunit * unit).mean(-1, keepdim=True))
    dh = dr * gate
    grads = [dr.to(s["x"].dtype), None, (dy * unit).reshape(-1, d).sum(0).to(s["weight"].dtype)]
    if s["post"] is not None:
        grads.append((dh * unit_h).reshape(-1, d).sum(0).to(s["post"].dtype))
        dunit_h = dh * s["post"].float()
        dbranch = rstd_h * (dunit_h - unit_h * (dunit_h * unit_h).mean(-1, keepdim=True))
    else:
        dbranch = dh
    grads[1] = dbranch.to(s["branch"].dtype)
    if s["gate"] is not None:
        dgate = dr * h * s["scale"]
        dgate = dgate.reshape(-1, d).sum(0) if s["gate"].dim() == 1 else dgate.sum(1, keepdim=True)
        grads.append(dgate.to(s["gate"].dtype))
    return (*first, *grads)


# ------------------------------------------------------------------ what it cannot do without
def work(case):
    if case["op"] == "attention":
        lengths = _lengths(case)
        rows = sum(lengths)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        whole = case["batch"] * case["tokens"]
        # a product of two matrices over the pairs: 2 in the forward, 5 more in the backward pass
        flops = (14 if case["backward"] else 4) * case["heads"] * pairs * case["dim"]
        wide, narrow = case["heads"] * case["dim"] * 2, case["kv_heads"] * case["dim"] * 2
        read = rows * (wide + 2 * narrow + (wide if case["backward"] else 0))
        written = whole * (wide + (wide + 2 * narrow if case["backward"] else 0))
        return {"bytes": read + written, "flops": flops}
    if case["op"] == "logprobs":
        n, size = case["rows"] * case["vocab"], TYPES[case["dtype"]].itemsize
        return {"bytes": n * size * (2 if case["backward"] else 1) + case["rows"] * (8 + 8 + 12 * case["top"] + (8 if case["backward"] else 0)),
                "flops": n * (10 if case["backward"] else 5)}
    n = case["batch"] * case["tokens"] * case["dim"]
    x, branch, out = (TYPES[case[name]].itemsize for name in ("x", "branch", "out"))
    moved = n * (2 * x + branch + out)
    if case["backward"]:  # the gradients of both outputs come in, those of both inputs go out
        moved += n * (2 * x + branch + out)
    vectors = case["dim"] * 4 * (1 + case["post"]) * (2 if case["backward"] else 1)
    return {"bytes": moved + vectors, "flops": n * (25 if case["backward"] else 8)}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"attention": _exact_attention, "logprobs": _exact_logprobs, "norm": _exact_norm}[case["op"]](s)


def _exact_attention(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    names = ("q", "k", "v")
    whole = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in names}
    o = torch.zeros_like(whole["q"])
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if case["causal"] else None
        for h in range(case["heads"]):  # one head at a time: the scores of a long sequence are large
            q = s["q"][i, h, :n].detach().double().requires_grad_()
            k = s["k"][i, h // group, :n].detach().double().requires_grad_()
            v = s["v"][i, h // group, :n].detach().double().requires_grad_()
            score = q @ k.t() / math.sqrt(case["dim"])
            if hidden is not None:
                score = score.masked_fill(hidden, -math.inf)
            out = torch.softmax(score, -1) @ v
            o[i, h, :n] = out.detach()
            if case["backward"]:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["do"][i, h, :n].double())
                whole["q"][i, h, :n] = dq
                whole["k"][i, h // group, :n] += dk
                whole["v"][i, h // group, :n] += dv
    return (o, *(whole[n] for n in names)) if case["backward"] else (o,)


def _exact_logprobs(s):
    case, parts = s["case"], []
    for at in range(0, case["rows"], 512):
        x = s["logits"][at:at + 512].detach().double().requires_grad_()
        tokens = s["tokens"][at:at + 512]
        lse = torch.logsumexp(x, -1)
        given = torch.gather(x, -1, tokens.clamp(min=0)[:, None])[:, 0] - lse
        logprob = torch.where(tokens < 0, torch.zeros_like(given), given)
        # H = lse - sum p x over the tokens that are allowed
        allowed = x.detach() > -math.inf
        p = torch.exp(x - lse[:, None])
        entropy = lse - (p * torch.where(allowed, x, torch.zeros_like(x))).sum(-1)
        out = [logprob.detach(), entropy.detach()]
        if case["backward"]:
            cotangents = s["dlogprob"][at:at + 512].double(), s["dentropy"][at:at + 512].double()
            out.append(torch.autograd.grad((logprob, entropy), x, cotangents)[0])
        elif case["top"]:
            best, ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True)
            out += [ids[:, :case["top"]].clone(), (best[:, :case["top"]] - lse[:, None]).detach()]
        parts.append(out)
    return tuple(torch.cat(column) for column in zip(*parts))


def _exact_norm(s):
    case = s["case"]
    names = [n for n in ("x", "branch", "weight", "post", "gate") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_() for n in names}

    def unit(z):
        return z / torch.sqrt((z * z).sum(-1, keepdim=True) / case["dim"] + EPS)

    h = unit(v["branch"]) * v["post"] if "post" in v else v["branch"]
    if "gate" in v:
        h = v["gate"] * h
    r = v["x"] + s["scale"] * h
    y = unit(r) * v["weight"]
    if not case["backward"]:
        return r.detach(), y.detach()
    grads = torch.autograd.grad((r, y), [v[n] for n in names], (s["dr"].double(), s["dy"].double()))
    return (r.detach(), y.detach(), *grads)
