"""Log probabilities of given tokens (with entropy and top alternatives) and distillation from a teacher's top
logits, as cases of a performance comparison: on given logits, and together with the LM head's product.

``run`` makes the calls of ``olmax_amd.ops`` where ``own`` is true.  Otherwise it computes the same in elementary torch
operations, in 32 bits whatever the inputs' type, rounded once at the end.  Vocabularies and widths are those of
``TransformerRecipe``; scores are z = cap(x) / temperature with cap(x) = softcap * tanh(x / softcap), p = softmax(z).
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
IGNORE = -100
VOCABS = [4096, 50304, 100278, 100352, 128256, 256000, 262144]
LOGITS_MOST = 4096 * 100352  # of the largest listed case on given logits


def _case(kind, **more):
    base = {"kind": kind, "dtype": "bf16", "top": 0, "temperature": 1.0, "softcap": 0.0, "padded": 0, "masked": 0}
    if kind.startswith("lmhead"):
        base["width"] = 4096
    if "distill" in kind:
        base |= {"top": 32, "tail": "renormalize", "grad": True}
    return {**base, **more}


def listed():
    return [
        # one token of one sequence, with the 20 alternatives that an interface shows: latency
        {"name": "score-1-token", **_case("score", tokens=1, vocab=128256, top=20)},
        # a batch of 37 continuations in fp32 logits, packed rows of a vocabulary that no vector length divides
        {"name": "score-37-f32", **_case("score", tokens=37, vocab=100278, dtype="f32", top=5, temperature=0.7)},
        # scoring a data set: every token of a 4096-token sequence, its entropy, no alternatives; 500 rows of padding
        {"name": "score-4096", **_case("score", tokens=4096, vocab=100352, padded=500)},
        # a teacher's pass that records its 64 best tokens, soft-capped logits over the largest vocabulary
        {"name": "score-teacher", **_case("score", tokens=1500, vocab=256000, top=64, softcap=30.0)},
        # policy gradient with an entropy bonus on a small model's logits
        {"name": "score-grad", **_case("score-grad", tokens=4096, vocab=50304, temperature=0.9, padded=100)},
        # the same in fp32 on few ragged rows, the vocabulary's last entries masked out
        {"name": "score-grad-f32", **_case("score-grad", tokens=333, vocab=100278, dtype="f32", masked=22)},
        # distillation in training: loss and gradient, the teacher's tail as one bucket
        {"name": "distill", **_case("distill", tokens=4096, vocab=100352, tail="bucket")},
        # evaluation against the teacher: loss alone, fp32 logits, many alternatives, softened
        {"name": "distill-loss", **_case("distill", tokens=700, vocab=128256, dtype="f32", top=128, temperature=2.0, grad=False)},
        # a handful of rows of the smallest vocabulary: launch latency
        {"name": "distill-9-rows", **_case("distill", tokens=9, vocab=4096, top=8)},
        # hidden states straight to log probabilities, no logits kept: a sequence of a 7B model
        {"name": "lmhead-score", **_case("lmhead-score", tokens=2048, vocab=100352)},
        # its gradients to the hidden states and to the LM head
        {"name": "lmhead-score-grad", **_case("lmhead-score-grad", tokens=1024, vocab=100352)},
        # distillation with the LM head in one call, a small model on a ragged batch
        {"name": "lmhead-distill", **_case("lmhead-distill", tokens=1500, vocab=50304, width=1024, top=64, tail="bucket")},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "score", "score", "score-grad", "score-grad", "distill", "distill", "lmhead-score", "lmhead-score-grad", "lmhead-distill"])
    V = rng.choice(VOCABS) if rng.random() < 0.7 else _log(rng, 1000, 262144)
    more = {"temperature": rng.choice([1.0, 1.0, 0.7, 2.0]), "softcap": rng.choice([0.0, 0.0, 30.0])}
    if "distill" in kind:
        more |= {"top": rng.choice([8, 32, 50, 64, 128]), "tail": rng.choice(["renormalize", "bucket"])}
    if kind.startswith("lmhead"):
        width = rng.choice([256, 1024, 4096, 4608])
        most = 2048 * 100352 * 4096 / (1 if kind == "lmhead-score" else 3)
        return _case(kind, tokens=max(1, min(_log(rng, 16, 2048), int(most / (width * V)))), vocab=V, width=width, **more)
    f32 = rng.random() < 0.4
    T = max(1, min(_log(rng, 1, 8192), LOGITS_MOST // V // (2 if f32 else 1)))
    if kind == "score":
        more["top"] = rng.choice([0, 1, 5, 20, 64, 128])
    if kind == "distill":
        more["grad"] = rng.random() < 0.7
    if kind != "distill":
        more["padded"] = T // 8 if rng.random() < 0.3 else 0
    return _case(kind, tokens=T, vocab=V, dtype="f32" if f32 else "bf16", masked=rng.choice([0, 0, V // 50]), **more)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, V, k = case["tokens"], case["vocab"], case["top"]
    dtype = F32 if case["dtype"] == "f32" else BF16
    normal = lambda *shape, std=1.0: torch.empty(*shape, device="cuda", dtype=F32).normal_(0.0, std, generator=gen)  # noqa: E731
    state = {"case": case}
    if case["kind"].startswith("lmhead"):
        d = case["width"]
        state["h"] = normal(T, d).to(BF16)  # behind the final norm
        state["w"] = normal(V, d, std=2.0 / math.sqrt(d)).to(BF16)
        z = None
    else:
        z = normal(T, V, std=2.5)
        sure = torch.rand(T, 1, device="cuda", generator=gen) * 14.0  # from undecided rows to sure ones
        best = torch.randint(0, V - case["masked"], (T, 1), device="cuda", generator=gen)
        z.scatter_add_(1, best, sure)
        if case["masked"]:
            z[:, V - case["masked"]:] = -math.inf
        state["logits"] = z.to(dtype)
    if "distill" in case["kind"]:
        # the teacher agrees with the student about much; from the hidden states its logits are not known: any tokens do
        if z is None:
            ids = torch.randint(0, V // k, (T, k), device="cuda", generator=gen) + torch.arange(k, device="cuda") * (V // k)
            t = normal(T, k, std=2.0)
            t = t - torch.logsumexp(t, 1, keepdim=True) - 0.2 * torch.rand(T, 1, device="cuda", generator=gen) - 0.02
        else:
            z = z * 0.8 + normal(T, V)
            t, ids = torch.topk(z, k, dim=1)
            t = t - torch.logsumexp(z, 1, keepdim=True)
        state["top_ids"], state["top_logprobs"] = ids.to(torch.int32), t.contiguous()
    else:
        targets = torch.randint(0, V - case["masked"], (T,), device="cuda", generator=gen)
        if z is not None:  # mostly what the row itself favours
            targets = torch.where(torch.rand(T, device="cuda", generator=gen) < 0.7, best[:, 0], targets)
        if case["padded"]:
            targets[T - case["padded"]:] = IGNORE
        state["targets"] = targets.to(torch.int32)
    if case["kind"].endswith("score-grad"):
        state["dlogprobs"] = normal(T)
        state["dentropy"] = normal(T, std=0.1)
        state["stats"] = _stats(state)
    return state


def _stats(state):
    """What a training step kept from its forward pass: (largest score, log of the sum of exponentials behind it, entropy) of each row."""
    case = state["case"]
    z = _scores(state["logits"] if "logits" in state else state["h"].float() @ state["w"].float().t(), case)
    m, log_sum, _, h = _rows(z)
    kept = state["targets"] != IGNORE
    return torch.stack([m, log_sum, h], 1) * kept[:, None]


def _scores(x, case):
    x = x.float()
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    return x / case["temperature"]


def _rows(z):
    """Largest score, log of the sum of exponentials behind it, probabilities and entropy of each row."""
    m = z.max(1).values
    z = z - m[:, None]
    e = torch.exp(z)
    s = e.sum(1)
    log_sum = torch.log(s)
    p = e / s[:, None]
    return m, log_sum, p, log_sum - torch.where(p > 0, p * z, 0.0).sum(1)


def _top_ids(x, k):
    """The k largest of each row in order, ties to the lowest index: whole numbers that rise with the value, and fall with the index."""
    V = x.shape[1]
    b = (x.float() + 0.0).view(torch.int32)
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b).to(torch.int64) * 2**32 + (V - 1 - torch.arange(V, device=x.device))
    return V - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)


def _plain_score(x, targets, case):
    z = _scores(x, case)
    m, log_sum, _, entropy = _rows(z)
    kept = targets != IGNORE
    at = torch.where(kept, targets, 0).long()[:, None]
    out = {"logprobs": torch.where(kept, z.gather(1, at)[:, 0] - m - log_sum, 0.0), "entropy": torch.where(kept, entropy, 0.0)}
    if case["top"]:
        ids = _top_ids(x, case["top"])
        out["top_logprobs"] = torch.where(kept[:, None], z.gather(1, ids) - (m + log_sum)[:, None], -math.inf)
        out["top_ids"] = torch.where(kept[:, None], ids, -1).to(torch.int32)
    return out


def _chain(x, case):
    """d z / d x."""
    c = case["softcap"]
    return (1.0 - torch.tanh(x.float() / c) ** 2 if c else 1.0) / case["temperature"]


def _plain_score_grad(x, state, case):
    kept = state["targets"] != IGNORE
    g, h = (torch.where(kept, state[n], 0.0)[:, None] for n in ("dlogprobs", "dentropy"))
    z = _scores(x, case)
    m, log_sum, p, entropy = _rows(z)
    logp = torch.where(p > 0, z - (m + log_sum)[:, None], 0.0)
    d = -p * (g + h * (logp + entropy[:, None]))
    d.scatter_add_(1, torch.where(kept, state["targets"], 0).long()[:, None], g)
    return d * _chain(x, case)


def _plain_distill(x, state, case, grad):
    ids, t = state["top_ids"].long(), state["top_logprobs"]
    z = _scores(x, case)
    m, log_sum, p, _ = _rows(z)
    logp = z.gather(1, ids) - (m + log_sum)[:, None]
    T = x.shape[0]
    if case["tail"] == "renormalize":
        t = t / case["temperature"]
        q = torch.exp(t - t.max(1, keepdim=True).values)
        q = q / q.sum(1, keepdim=True)
        loss = (q * (torch.log(q) - logp)).sum(1)
        d = p
    else:
        q = torch.exp(t)
        rest = p.scatter(1, ids, 0.0).sum(1)
        r = (1.0 - q.sum(1)).clamp(min=0.0)
        loss = (q * (t - logp)).sum(1) + torch.where(r > 0, r * torch.log(r / rest), 0.0)
        d = (p * (1.0 - r / rest)[:, None]).scatter(1, ids, p.gather(1, ids))
    if not grad:
        return loss.mean(), None
    d = d.scatter_add(1, ids, -q) * _chain(x, case) / T
    return loss.mean(), d


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from olmax_amd import ops

        kw = {"temperature": case["temperature"], "softcap": case["softcap"]}
        if kind == "score":
            r = ops.token_logprobs(state["logits"], state["targets"], top=case["top"], ignore_index=IGNORE, **kw)
            out = {"logprobs": r.logprobs, "entropy": r.entropy}
            return {**out, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids} if case["top"] else out
        if kind == "score-grad":
            return ops.token_logprobs_bwd(state["logits"], state["targets"], state["stats"], state["dlogprobs"], dentropy=state["dentropy"],
                                          ignore_index=IGNORE, **kw)
        if kind == "distill":
            loss, d = ops.distill(state["logits"], state["top_ids"], state["top_logprobs"], tail=case["tail"], want_grad=case["grad"], **kw)
            return {"loss": loss, "dlogits": d} if case["grad"] else loss
        if kind == "lmhead-score":
            r = ops.lmhead_logprobs(state["h"], state["w"], state["targets"], ignore_index=IGNORE, **kw)
            return {"logprobs": r.logprobs, "entropy": r.entropy}
        if kind == "lmhead-score-grad":
            dh, dw = ops.lmhead_logprobs_bwd(state["h"], state["w"], state["targets"], state["stats"], state["dlogprobs"],
                                             dentropy=state["dentropy"], ignore_index=IGNORE, **kw)
            return {"dh": dh, "dw": dw}
        loss, dh, dw = ops.lmhead_distill(state["h"], state["w"], state["top_ids"], state["top_logprobs"], tail=case["tail"], **kw)
        return {"loss": loss, "dh": dh, "dw": dw}
    if kind == "score":
        return _plain_score(state["logits"], state["targets"], case)
    if kind == "score-grad":
        return _plain_score_grad(state["logits"], state, case).to(state["logits"].dtype)
    if kind == "distill":
        loss, d = _plain_distill(state["logits"], state, case, case["grad"])
        return {"loss": loss, "dlogits": d.to(state["logits"].dtype)} if case["grad"] else loss
    h, w = state["h"].float(), state["w"].float()
    x = h @ w.t()
    if kind == "lmhead-score":
        return _plain_score(x, state["targets"], case)
    if kind == "lmhead-score-grad":
        d = _plain_score_grad(x, state, case)
        return {"dh": (d @ w).to(BF16), "dw": (d.t() @ h).to(BF16)}
    loss, d = _plain_distill(x, state, case, True)
    return {"loss": loss, "dh": (d @ w).to(BF16), "dw": (d.t() @ h).to(BF16)}


def exact(case, seed):
    """From the definitions in 64 bits: -KL, log-softmax and entropy, and gradients as the sums over outputs of cotangent times derivative."""
    state = prepare(case, seed)
    head = case["kind"].startswith("lmhead")
    h, w = (state["h"].double(), state["w"].double()) if head else (None, None)
    x = h @ w.t() if head else state["logits"].double()
    T, V = x.shape
    cap, tau = case["softcap"], case["temperature"]
    slope = torch.full_like(x, 1 / tau) if not cap else 1 / (torch.cosh(x / cap) ** 2 * tau)
    y = x / tau if not cap else torch.tanh(x / cap) * (cap / tau)
    logp = y - torch.logsumexp(y, 1, keepdim=True)
    del y
    prob = logp.exp()
    rows = torch.arange(T, device=x.device)
    if "distill" in case["kind"]:
        ids, t = state["top_ids"].long(), state["top_logprobs"].double()
        inside = torch.zeros(T, V, dtype=torch.bool, device=x.device)
        inside[rows[:, None], ids] = True
        if case["tail"] == "renormalize":
            q = torch.softmax(t / tau, 1)
            loss = (torch.xlogy(q, q) - q * logp.gather(1, ids)).sum(1)
            outside = 1.0
        else:
            q = t.exp()
            r = (1 - q.sum(1)).clamp(min=0)
            s = torch.where(inside, 0.0, prob).sum(1)
            loss = (q * (t - logp.gather(1, ids))).sum(1) + torch.xlogy(r, r) - torch.xlogy(r, s)
            outside = ((s - r) / s)[:, None]
        out = {"loss": loss.mean()}
        if not case["grad"]:
            return out["loss"]
        d = torch.where(inside, prob, prob * outside)
        d[rows[:, None], ids] -= q
        d *= slope / T
        return {**out, "dh": d @ w, "dw": d.t() @ h} if head else {**out, "dlogits": d}
    kept = state["targets"] != IGNORE
    at = state["targets"].long().clamp(min=0)
    plogp = torch.where(prob > 0, prob * logp, 0.0)
    entropy = -plogp.sum(1)
    if case["kind"].endswith("score"):
        out = {"logprobs": logp[rows, at] * kept, "entropy": entropy * kept}
        if case["top"]:
            best = torch.topk(logp, case["top"], dim=1).values
            out |= {"top_logprobs": torch.where(kept[:, None], best, -math.inf), "top_ids": None}
        return out
    g, e = ((state[n].double() * kept)[:, None] for n in ("dlogprobs", "dentropy"))
    d = -g * prob - e * (plogp + prob * entropy[:, None])
    d[rows, at] += g[:, 0]
    d *= slope
    return {"dh": d @ w, "dw": d.t() @ h} if head else d


def work(case):
    T, V, k = case["tokens"], case["vocab"], case["top"]
    kept = T - case["padded"]
    size = 4 if case["dtype"] == "f32" else 2
    given = 12.0 * T + 8.0 * T * k  # a row's numbers, and its alternatives
    # sub, exp, two sums, product of each logit forward; about as much again for its gradient
    if case["kind"] == "score":
        return {"bytes": kept * V * size + given, "flops": 5.0 * kept * V}
    if case["kind"] == "score-grad":
        return {"bytes": (kept + T) * V * size + given, "flops": 6.0 * kept * V}
    if case["kind"] == "distill":
        return {"bytes": T * V * size * (2 if case["grad"] else 1) + given, "flops": (10.0 if case["grad"] else 5.0) * T * V}
    d = case["width"]
    products = 1 if case["kind"] == "lmhead-score" else 3
    return {"bytes": 2.0 * (T + V) * d * (1 if products == 1 else 2) + given, "flops": products * 2.0 * T * V * d + 5.0 * T * V}
