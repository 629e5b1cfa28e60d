"""Cases that measure the vocabulary operators: token log-probabilities (with entropies and top
alternatives), distillation from a teacher's top tokens, and both straight from hidden states.

With ``own`` unset ``run`` computes the plain form in elementary fp32 torch operations; with it set
it makes the calls a user makes of :mod:`ohara_b200.ops`. ``exact`` states the same definitions in
64 bits (gradients by autograd there, by formula in the plain form).
"""

import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------------------
def _logprobs(name, rows, vocab, dtype, top, entropy, grad, temperature=1.0, ignored=0.0,
              masked=0.0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "entropy": entropy, "grad": grad, "temperature": temperature, "ignored": ignored,
            "masked": masked}


def _distill(name, rows, vocab, dtype, top, tail, temperature=1.0):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "tail": tail, "grad": True, "temperature": temperature}


def _linear_logprobs(name, rows, hidden, vocab, entropy, grad, temperature=1.0, ignored=0.0):
    return {"name": name, "op": "linear_logprobs", "rows": rows, "hidden": hidden, "vocab": vocab,
            "entropy": entropy, "grad": grad, "temperature": temperature, "ignored": ignored}


def _linear_distill(name, rows, hidden, vocab, top, tail, temperature=1.0):
    return {"name": name, "op": "linear_distill", "rows": rows, "hidden": hidden, "vocab": vocab,
            "top": top, "tail": tail, "grad": True, "temperature": temperature}


def listed():
    return [
        # one sequence being decoded: the sampled token's log-probability and 20 alternatives
        _logprobs("decode_1", 1, 50304, "bf16", 20, True, False),
        # a full serving batch with constrained decoding: a tenth of the vocabulary masked out
        _logprobs("decode_64_masked", 64, 50304, "bf16", 5, False, False, masked=0.1),
        # scoring four packed sequences (evaluation): the targets' log-probability and the best token
        _logprobs("score_8188", 4 * 2047, 50304, "bf16", 1, False, False, ignored=0.25),
        # writing a teacher's 64 best tokens at temperature 2 for later distillation
        _logprobs("teacher_top64", 4096, 131072, "bf16", 64, False, False, temperature=2.0),
        # a preference / policy-gradient step: fp32 logits of an unpadded vocabulary, with entropy
        _logprobs("policy_step_odd", 2047, 50257, "fp32", 0, True, True),
        # distillation of a small model on a short batch
        _distill("distill_small", 130, 8192, "fp32", 8, False),
        # distillation on packed sequences; mass outside the teacher's list in a bucket of its own
        _distill("distill_tail", 4 * 2047, 50304, "bf16", 32, True, temperature=2.0),
        # the same step at the depth-12 model's batch, list renormalised
        _distill("distill_large", 16384, 50304, "bf16", 64, False),
        # log-probabilities of one short reply straight from the final hidden states
        _linear_logprobs("reply_37", 37, 768, 50304, False, False),
        # preference step of the depth-12 model without stored logits
        _linear_logprobs("policy_step_hidden", 4 * 2047, 768, 50304, True, True, ignored=0.25),
        # distillation into the 1.3B-wide head, one short sequence
        _linear_distill("distill_hidden_500", 500, 2048, 50304, 16, True),
        # distillation into the depth-16 width, packed sequences
        _linear_distill("distill_hidden_4096", 4096, 1024, 50304, 32, False, temperature=2.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "distill", "distill", "linear_logprobs", "linear_distill"])
    vocab = _log_int(rng, 8192, 131072)
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op == "logprobs":
        rows = _log_int(rng, 1, min(8192, 400_000_000 // vocab))
        grad = rng.random() < 0.5
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "top": 0 if grad else rng.choice([0, 1, _log_int(rng, 2, 64)]),
                "entropy": rng.random() < 0.5, "grad": grad, "temperature": temperature,
                "ignored": rng.choice([0.0, 0.25]), "masked": 0.0 if grad else rng.choice([0.0, 0.1])}
    if op == "distill":
        rows = _log_int(rng, 1, min(8192, 400_000_000 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "top": _log_int(rng, 1, 64), "tail": rng.random() < 0.5, "grad": True,
                "temperature": temperature}
    rows = _log_int(rng, 1, min(4096, 200_000_000 // vocab))
    case = {"op": op, "rows": rows, "hidden": 8 * _log_int(rng, 32, 256), "vocab": vocab,
            "temperature": temperature}
    if op == "linear_logprobs":
        return {**case, "entropy": rng.random() < 0.5, "grad": rng.random() < 0.5,
                "ignored": rng.choice([0.0, 0.25])}
    return {**case, "top": _log_int(rng, 1, 64), "tail": rng.random() < 0.5, "grad": True}


# --------------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 17)
    return gen


def _tokens(gen, rows, vocab, ignored):
    """Target tokens, the frequent (low) ids more often; a share of the rows is prompt."""
    u = torch.rand(rows, device="cuda", generator=gen)
    tokens = (vocab ** u).long().clamp_(1, vocab) - 1
    if ignored > 0:
        drop = torch.rand(rows, device="cuda", generator=gen) < ignored
        tokens = tokens.masked_fill(drop, IGNORE)
    return tokens


def _logits(gen, rows, vocab, dtype, tokens):
    """A language model's logits: a frequency profile over the ids, noise for the context, and a
    lift of the token that comes next."""
    profile = -torch.log1p(torch.arange(vocab, device="cuda", dtype=torch.float32) * 0.02)
    x = torch.empty(rows, vocab, device="cuda", dtype=dtype)
    step = max(1, 128_000_000 // vocab)
    for begin in range(0, rows, step):
        part = torch.randn(min(step, rows - begin), vocab, device="cuda", generator=gen)
        part.mul_(1.8).add_(profile)
        at = tokens[begin:begin + step].clamp_min(0).unsqueeze(1)
        part.scatter_add_(1, at, torch.full_like(at, 4.0, dtype=torch.float32))
        x[begin:begin + step] = part
    return x


def _teacher(gen, rows, vocab, top, tokens):
    """A teacher's list per row: the next token and others (each once), their log-probabilities
    with some mass left outside; the last entries of every ninth row are padding."""
    # distinct ids: the target plus multiples of a stride that is no divisor of the vocabulary
    stride = max(1, vocab // (top + 1))
    others = torch.arange(top, device="cuda") * stride
    listed_tokens = (tokens.clamp_min(0).unsqueeze(1) + others) % vocab
    scores = 2.0 * torch.randn(rows, top, device="cuda", generator=gen)
    scores[:, 0] += 4.0
    outside = 1.5 * torch.randn(rows, 1, device="cuda", generator=gen)
    logprobs = torch.log_softmax(torch.cat([scores, outside], dim=1), dim=1)[:, :-1].contiguous()
    if top > 1:
        listed_tokens[::9, top - (top + 3) // 4:] = -1
    return logprobs, listed_tokens


def prepare(case, seed):
    gen = _generator(seed)
    rows, vocab, op = case["rows"], case["vocab"], case["op"]
    state = {"case": dict(case)}
    tokens = _tokens(gen, rows, vocab, case.get("ignored", 0.0))
    if op.startswith("linear"):
        hidden = torch.randn(rows, case["hidden"], device="cuda", generator=gen)
        weight = torch.randn(vocab, case["hidden"], device="cuda", generator=gen)
        weight.mul_(2.0 / math.sqrt(case["hidden"]))
        state["hidden"] = hidden.bfloat16().requires_grad_(case["grad"])
        state["weight"] = weight.bfloat16().requires_grad_(case["grad"])
    else:
        logits = _logits(gen, rows, vocab, DTYPES[case["dtype"]], tokens)
        if case.get("masked", 0.0) > 0:
            out = torch.rand(vocab, device="cuda", generator=gen) < case["masked"]
            logits.masked_fill_(out, -math.inf)
        state["logits"] = logits.requires_grad_(case["grad"])
    if op.endswith("distill"):
        state["teacher_logprobs"], state["teacher_tokens"] = _teacher(gen, rows, vocab, case["top"],
                                                                      tokens)
    else:
        state["tokens"] = tokens
    if case["grad"]:
        scale = 1.0 / max(rows, 1)
        state["d_out"] = scale * (1.0 + torch.rand(rows, device="cuda", generator=gen))
        state["d_entropy"] = -0.3 * scale * (1.0 + torch.rand(rows, device="cuda", generator=gen))
    return state


# --------------------------------------------------------------------------------------------------
# The framework's calls
# --------------------------------------------------------------------------------------------------
def _own(state):
    from ohara_b200 import ops

    case = state["case"]
    op, temperature = case["op"], case["temperature"]
    leaves = [state["hidden"], state["weight"]] if op.startswith("linear") else [state["logits"]]
    out, heads, upstream = {}, [], []
    if op.endswith("distill"):
        fn = ops.linear_distillation_loss if op.startswith("linear") else ops.distillation_loss
        loss = fn(*leaves, state["teacher_logprobs"], state["teacher_tokens"],
                  temperature=temperature, tail=case["tail"])
        out["loss"] = loss
        heads, upstream = [loss], [state["d_out"]] if case["grad"] else []
    else:
        fn = ops.linear_token_logprobs if op.startswith("linear") else ops.token_logprobs
        got = fn(*leaves, state["tokens"], temperature=temperature, entropy=case["entropy"],
                 top=case.get("top", 0), ignore_index=IGNORE)
        out["logprobs"] = got.logprobs
        heads, upstream = [got.logprobs], [state["d_out"]] if case["grad"] else []
        if case["entropy"]:
            out["entropy"] = got.entropy
            heads.append(got.entropy)
            upstream += [state["d_entropy"]] if case["grad"] else []
        if case.get("top", 0):
            out["top_logprobs"], out["top_tokens"] = got.top_logprobs, got.top_tokens
    if case["grad"]:
        for name, grad in zip(("d_first", "d_weight"), torch.autograd.grad(heads, leaves, upstream)):
            out[name] = grad
    return out


# --------------------------------------------------------------------------------------------------
# The plain form, 32 bits
# --------------------------------------------------------------------------------------------------
def _softmax_parts(logits, temperature):
    """``(log q, q)`` of fp32 scaled logits."""
    z = logits / temperature
    z = z - z.amax(dim=1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(dim=1, keepdim=True)
    return z - torch.log(total), e / total


def _plain_logprobs(logits, state, out):
    """Outputs of token log-probabilities and, with gradients, d(loss) / d(logits)."""
    case, tokens = state["case"], state["tokens"]
    temperature = case["temperature"]
    keep = tokens != IGNORE
    at = tokens.masked_fill(~keep, 0).unsqueeze(1)
    logq, q = _softmax_parts(logits, temperature)
    zero = torch.zeros((), device=logits.device)
    out["logprobs"] = torch.where(keep, logq.gather(1, at).squeeze(1), zero)
    entropy = None
    if case["entropy"]:
        entropy = -torch.where(q > 0, q * logq, zero).sum(dim=1)
        out["entropy"] = torch.where(keep, entropy, zero)
    if case.get("top", 0):
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_logprobs"] = torch.where(keep.unsqueeze(1), logq.gather(1, order),
                                          torch.full((), -math.inf, device=logits.device))
        out["top_tokens"] = order.masked_fill(~keep.unsqueeze(1), -1)
    if not case["grad"]:
        return None
    g = torch.where(keep, state["d_out"], zero).unsqueeze(1)
    d = -q * g
    d.scatter_add_(1, at, g)
    if entropy is not None:
        ge = torch.where(keep, state["d_entropy"], zero).unsqueeze(1)
        d -= ge * q * (logq + entropy.unsqueeze(1))
    return d / temperature


def _plain_distill(logits, state, out):
    case = state["case"]
    temperature = case["temperature"]
    entry, values = state["teacher_tokens"], state["teacher_logprobs"]
    present = entry >= 0
    at = entry.clamp_min(0)
    zero = torch.zeros((), device=logits.device)
    logq, q = _softmax_parts(logits, temperature)
    if case["tail"]:
        p = torch.where(present, torch.exp(values), zero)
        logp = values
    else:
        peak = torch.where(present, values, torch.full_like(values, -math.inf)).amax(1, keepdim=True)
        p = torch.where(present, torch.exp(values - peak), zero)
        total = p.sum(dim=1, keepdim=True)
        p = p / total
        logp = values - peak - torch.log(total)
    picked = logq.gather(1, at)
    loss = torch.where(present, p * (logp - picked), zero).sum(dim=1)
    weight = torch.ones_like(loss).unsqueeze(1)
    if case["tail"]:
        inside = torch.zeros(logits.shape, device=logits.device)
        inside.scatter_add_(1, at, present.float())
        outside = inside == 0
        qt = torch.where(outside, q, zero).sum(dim=1, keepdim=True)
        listed_mass = p.sum(dim=1, keepdim=True)
        pt = (1.0 - listed_mass).clamp_min(0.0)
        some = pt > 0
        loss = loss + torch.where(some, pt * (torch.log(pt.clamp_min(1e-38)) - torch.log(qt)),
                                  zero).squeeze(1)
        weight = listed_mass + pt
    out["loss"] = loss
    d = q * weight
    if case["tail"]:
        d = d - torch.where(outside, q, zero) * torch.where(some, pt / qt, zero)
    d.scatter_add_(1, at, torch.where(present, -p, zero))
    return d * (state["d_out"].unsqueeze(1) / temperature)


def _plain(state):
    case, out = state["case"], {}
    linear = case["op"].startswith("linear")
    if linear:
        hidden, weight = state["hidden"].detach().float(), state["weight"].detach().float()
        logits = hidden @ weight.T
    else:
        logits = state["logits"].detach().float()
    d = (_plain_distill if case["op"].endswith("distill") else _plain_logprobs)(logits, state, out)
    if case["grad"]:
        if linear:
            out["d_first"] = (d @ weight).to(state["hidden"].dtype)
            out["d_weight"] = (d.T @ hidden).to(state["weight"].dtype)
        else:
            out["d_first"] = d.to(state["logits"].dtype)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------------------------------
def _exact_rows(logits, state, rows):
    """Values (and the scalar whose gradient is asked for) of a slice of rows; logits are fp64."""
    case = state["case"]
    logq = torch.log_softmax(logits / case["temperature"], dim=1)
    got, scalar = {}, 0.0
    if case["op"].endswith("distill"):
        entry = state["teacher_tokens"][rows]
        values = state["teacher_logprobs"][rows].double()
        values = values.masked_fill(entry < 0, -math.inf)
        logp = values if case["tail"] else torch.log_softmax(values, dim=1)
        keep = entry >= 0
        terms = logp.exp() * (logp.masked_fill(~keep, 0.0) - logq.gather(1, entry.clamp_min(0)))
        loss = terms.masked_fill(~keep, 0.0).sum(dim=1)
        if case["tail"]:
            pt = -torch.expm1(torch.logsumexp(values, dim=1))
            listed_ids = entry.masked_fill(~keep, logits.shape[1])
            hidden_part = torch.cat([logq, logq.new_full((len(logq), 1), -math.inf)], dim=1)
            rest = torch.logsumexp(hidden_part.scatter(1, listed_ids, -math.inf), dim=1)
            loss = loss + pt * (pt.log() - rest)
        got["loss"] = loss
        if case["grad"]:
            scalar = (loss * state["d_out"][rows].double()).sum()
    else:
        tokens = state["tokens"][rows]
        keep = tokens != IGNORE
        l = logq.gather(1, tokens.masked_fill(~keep, 0).unsqueeze(1)).squeeze(1).masked_fill(~keep, 0.0)
        got["logprobs"] = l
        if case["grad"]:
            scalar = (l * state["d_out"][rows].double()).sum()
        if case["entropy"]:
            finite = logq.masked_fill(logq == -math.inf, 0.0)
            h = -(logq.exp() * finite).sum(dim=1).masked_fill(~keep, 0.0)
            got["entropy"] = h
            if case["grad"]:
                scalar = scalar + (h * state["d_entropy"][rows].double()).sum()
        if case.get("top", 0):
            best = logq.topk(case["top"], dim=1).values
            got["top_logprobs"] = best.masked_fill(~keep.unsqueeze(1), -math.inf)
    return got, scalar


def exact(case, seed):
    state = prepare(case, seed)
    linear = case["op"].startswith("linear")
    n, vocab = case["rows"], case["vocab"]
    step = max(1, 64_000_000 // vocab)
    parts, d_rows, d_weight = [], [], None
    if linear:
        weight = state["weight"].detach().double()
        d_weight = torch.zeros_like(weight)
    for begin in range(0, n, step):
        rows = slice(begin, min(begin + step, n))
        if linear:
            hidden = state["hidden"].detach()[rows].double()
            logits = hidden @ weight.T
        else:
            logits = state["logits"].detach()[rows].double()
        logits.requires_grad_(case["grad"])
        with torch.enable_grad():
            got, scalar = _exact_rows(logits, state, rows)
        parts.append({k: v.detach() for k, v in got.items()})
        if case["grad"]:
            (d,) = torch.autograd.grad(scalar, logits)
            if linear:
                d_rows.append(d @ weight)
                d_weight.addmm_(d.T, hidden)
            else:
                d_rows.append(d)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case.get("top", 0) and case["op"] == "logprobs":
        out["top_tokens"] = None
    if case["grad"]:
        out["d_first"] = torch.cat(d_rows)
        if linear:
            out["d_weight"] = d_weight
    return out


# --------------------------------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    rows, vocab = case["rows"], case["vocab"]
    used = rows * (1.0 - case.get("ignored", 0.0))
    top = case.get("top", 0)
    per_logit = 8.0 + (4.0 if case.get("entropy") else 0.0) + (6.0 if case["grad"] else 0.0)
    small = rows * (8.0 + 4.0 + (4.0 if case.get("entropy") else 0.0) + 12.0 * top)
    if not case["op"].startswith("linear"):
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        read = used * vocab * size
        write = rows * vocab * size if case["grad"] else 0.0
        return {"bytes": read + write + small, "flops": used * vocab * per_logit}
    d = case["hidden"]
    products = 3.0 if case["grad"] else 1.0
    move = 2.0 * (rows * d + vocab * d) * (2.0 if case["grad"] else 1.0)
    return {"bytes": move + small, "flops": 2.0 * used * d * vocab * products + used * vocab * per_logit}
