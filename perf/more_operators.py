"""Rotary positions (tables scaled for long contexts, half and interleaved pairs, part of a head, given positions) with their gradient, and
differential attention, the difference of two softmax maps with a learned weight, with its gradients, as cases of a performance comparison.

``run`` makes the calls of ``olmax_amd.ops`` where ``own`` is true.  Otherwise it computes the same in elementary torch operations, in 32 bits
whatever the inputs' type (angles in 64), rounded once at the end.  Heads, widths, windows and lengths are those of ``TransformerRecipe``.

Tables: angle(p, i) = p f_i, f_i = theta^(-2i/R) slowed down as the scaling says.  Rotation of a pair (a, b) by it: (a cos - b sin, b cos + a sin);
pairs are (i, i + R/2) in the half layout and (2i, 2i + 1) in the interleaved one; columns of a head from R on pass.

Attention: a query head h has two queries and its key head two keys of width D, and values of width 2D.  With P_m the causal softmax of
q_m k_m^T / sqrt(D), o = (P_1 - lambda_h P_2) v.  The two queries of a head lie side by side in a row, and so do the keys.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
PAIRS_FORWARD, PAIRS_BACKWARD = 2 * 32 * 4096**2, 32 * 4096**2  # of the largest listed attention (query, key, head), masked ones among them
ROTATED = 8192 * 64 * 128  # values of the largest listed rotation


def _tables(**more):
    return {"kind": "tables", "theta": 500000.0, "scaling": "none", "factor": 1.0, "original": 8192, **more}


def _rotate(**more):
    return {"kind": "rotate", "dtype": "bf16", "head_dim": 128, "layout": "half", "seq": 0, "padded": 0, "spare": 0, **more}


def _attn(kind, **more):
    return {"kind": kind, "window": -1, "shared": False, **more}


def listed():
    return [
        # a model of 8192 tokens' context carried to 131072: done once, when it is loaded
        {"name": "tables-131072", **_tables(length=131072, rotary=128, scaling="llama3", factor=8.0)},
        # the same for a small model, four times its context
        {"name": "tables-yarn", **_tables(length=16384, rotary=64, theta=10000.0, scaling="yarn", factor=4.0, original=4096)},
        # one token of one sequence, far out in the context, queries and keys of 32 / 8 heads: latency
        {"name": "rotate-1-token", **_rotate(tokens=1, heads=40, rotary=128)},
        # queries and keys of a 7B model's step (2 x 4096 tokens), out of the rows that the fused projection leaves
        {"name": "rotate-8192", **_rotate(tokens=8192, heads=64, rotary=128, seq=4096, spare=32)},
        # interleaved pairs, half of each head, documents packed in a ragged batch, the last tokens padding
        {"name": "rotate-part", **_rotate(tokens=5001, heads=48, rotary=64, layout="interleaved", padded=300)},
        # the gradient, on the two queries and keys of 64 that differential attention has in the place of one of 128
        {"name": "rotate-grad", **_rotate(kind="rotate-grad", tokens=4096, heads=128, head_dim=64, rotary=64, seq=4096)},
        # a small model on a short prompt: latency
        {"name": "diff-100", **_attn("diff", batch=1, seq=100, heads=4, kv_heads=4, dim=32)},
        # a 7B model's training step, forward
        {"name": "diff-4096", **_attn("diff", batch=2, seq=4096, heads=32, kv_heads=32, dim=64)},
        # a layer with a window, two query heads to a key head, ragged length
        {"name": "diff-window", **_attn("diff", batch=1, seq=4001, heads=32, kv_heads=16, dim=64, window=1024)},
        # a small model's gradients on short ragged sequences, one weight for all heads
        {"name": "diff-grad-333", **_attn("diff-grad", batch=3, seq=333, heads=4, kv_heads=2, dim=32, shared=True)},
        # gradients at 4096 tokens, four query heads to a key head
        {"name": "diff-grad-4096", **_attn("diff-grad", batch=1, seq=4096, heads=32, kv_heads=8, dim=64)},
        # gradients of a layer with a window
        {"name": "diff-grad-window", **_attn("diff-grad", batch=1, seq=5000, heads=16, kv_heads=8, dim=64, window=1024)},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rotate", "rotate", "rotate", "rotate-grad", "diff", "diff", "diff", "diff-grad", "diff-grad", "diff-grad"])
    if kind == "tables":
        scaling = rng.choice(["none", "linear", "llama3", "yarn"])
        return _tables(length=_log(rng, 100, 131072), rotary=rng.choice([32, 64, 128]), theta=rng.choice([1e4, 5e5, 1e6]), scaling=scaling,
                       factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), original=rng.choice([4096, 8192]))
    if kind.startswith("rotate"):
        dim = rng.choice([64, 128])
        heads = rng.choice([4, 5, 12, 40, 48, 64, 128])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        tokens = min(_log(rng, 1, 16384), ROTATED // (heads * dim) // (2 if dtype == "f32" else 1))
        return _rotate(kind=kind, tokens=tokens, heads=heads, head_dim=dim, rotary=rng.choice([dim, dim, dim // 2, dim // 4]), dtype=dtype,
                       layout=rng.choice(["half", "interleaved"]), seq=rng.choice([0, 1 + tokens // 2]), padded=rng.choice([0, tokens // 9]), spare=rng.choice([0, 0, 3, heads // 2]))
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 2, 4])
    most = PAIRS_BACKWARD if kind == "diff-grad" else PAIRS_FORWARD
    batch = rng.choice([1, 1, 2, 3])
    seq = max(1, min(_log(rng, 1, 8192), int(math.sqrt(most / (batch * heads)))))
    return _attn(kind, batch=batch, seq=seq, heads=heads, kv_heads=kv, dim=rng.choice([32, 64, 64]), window=rng.choice([-1, -1, 1024, seq // 3]), shared=rng.random() < 0.3)


# ----------------------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, std=1.0: torch.empty(*shape, device="cuda", dtype=F32).normal_(0.0, std, generator=gen)  # noqa: E731
    state = {"case": case}
    if case["kind"] == "tables":  # nothing but numbers go in: a new state has another base
        state["theta"] = case["theta"] * (1.0 + (seed % 1009) / 1009.0)
    elif case["kind"].startswith("rotate"):
        T, heads, D, R = case["tokens"], case["heads"], case["head_dim"], case["rotary"]
        dtype = F32 if case["dtype"] == "f32" else BF16
        state["x"] = normal(T, (heads + case["spare"]) * D).to(dtype)[:, : heads * D]
        length = max(T, 4096) if case["seq"] else 131072  # places that the tables have
        angle = torch.arange(length, device="cuda", dtype=F64)[:, None] * 500000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=F64) / R)
        state["cos"], state["sin"] = angle.cos().to(F32), angle.sin().to(F32)
        if case["seq"]:
            state["positions"] = None  # every row's place in its sequence
        else:  # documents of some hundred tokens, one behind the other; the first begins anywhere
            starts = (torch.rand(T, device="cuda", generator=gen) < 1 / 300).long()
            at = torch.arange(T, device="cuda")
            begin = torch.cummax(torch.where(starts > 0, at, 0), 0).values
            first = torch.randint(0, length - T + 1, (1,), device="cuda", generator=gen)
            state["positions"] = torch.where(begin == 0, at + first, at - begin).to(torch.int32)
            if case["padded"]:
                state["positions"][T - case["padded"]:] = -1
    else:
        B, S, H, KH, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
        # scores of a trained head: some keys stand out
        state["q"] = normal(B * S, H * 2 * D, std=1.5).to(BF16)
        state["k"] = normal(B * S, KH * 2 * D, std=1.5).to(BF16)
        state["v"] = normal(B * S, KH * 2 * D).to(BF16)
        state["lam"] = 0.2 + 0.5 * torch.rand(1 if case["shared"] else H, device="cuda", generator=gen)
        if case["kind"] == "diff-grad":
            state["do"] = normal(B * S, H * 2 * D).to(BF16)
            # kept from the forward pass: its outputs, the second map's, and both maps' log-normalisers
            o, o2, lse = _plain_diff(state)
            state |= {"o": o, "o2": o2, "lse": lse}
    return state


# ----------------------------------------------------------------------------- plain forms
def _plain_tables(theta, case, device):
    R, L, s = case["rotary"], float(case["original"]), case["factor"]
    i = torch.arange(R // 2, device=device, dtype=F64)
    f = theta ** (-2.0 * i / R)
    size = 1.0
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "llama3":  # waves that fit the original context less than once are slowed down, those that fit four times are not
        fits = L * f / (2.0 * math.pi)
        keep = ((fits - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / s
    elif case["scaling"] == "yarn":  # by the index: a ramp from where 32 waves fit to where one does
        at = lambda turns: R * math.log(L / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), R - 1)
        slow = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        f = f * (1.0 - slow) + f / s * slow
        size = 0.1 * math.log(s) + 1.0
    angle = torch.arange(case["length"], device=device, dtype=F64)[:, None] * f
    return (angle.cos() * size).to(F32), (angle.sin() * size).to(F32)


def _positions(state):
    case = state["case"]
    if state["positions"] is not None:
        return state["positions"].long()
    return torch.arange(case["tokens"], device=state["x"].device) % case["seq"]


def _plain_rotate(state, sign):
    case, x = state["case"], state["x"]
    T, heads, D, R = case["tokens"], case["heads"], case["head_dim"], case["rotary"]
    p = _positions(state)
    at = p.clamp(min=0)
    c, s = state["cos"][at][:, None, :], sign * state["sin"][at][:, None, :]
    xf = x.float().view(T, heads, D)
    if case["layout"] == "half":
        a, b = xf[..., : R // 2], xf[..., R // 2: R]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = xf[..., 0:R:2], xf[..., 1:R:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    y = torch.cat([turned, xf[..., R:]], -1)
    return torch.where((p < 0)[:, None, None], xf, y).view(T, heads * D).to(x.dtype)


def _seen(case, device):
    """[S, S]: whether the query of a row sees the key of a column."""
    at = torch.arange(case["seq"], device=device)
    far = at[:, None] - at[None, :]
    return (far >= 0) & (far <= case["window"]) if case["window"] >= 0 else far >= 0


def _split(t, case, groups):
    """[B S, heads 2 width] as [B, kv heads, query heads to each (groups) or 1, 2, S, width], fp32."""
    B, S, KH = case["batch"], case["seq"], case["kv_heads"]
    return t.float().view(B, S, KH, groups, 2, -1).permute(0, 2, 3, 4, 1, 5)


def _join(t, case):
    return t.permute(0, 4, 1, 2, 3, 5).reshape(case["batch"] * case["seq"], -1)


def _values(t, case, groups):
    """[B S, heads 2D] as [B, kv heads, groups, S, 2D], fp32."""
    B, S, KH = case["batch"], case["seq"], case["kv_heads"]
    return t.float().view(B, S, KH, groups, -1).permute(0, 2, 3, 1, 4)


def _rows(t, case):
    return t.permute(0, 3, 1, 2, 4).reshape(case["batch"] * case["seq"], -1)


def _plain_scores(state):
    case = state["case"]
    q, k = _split(state["q"], case, case["heads"] // case["kv_heads"]), _split(state["k"], case, 1)
    return (torch.matmul(q, k.transpose(-1, -2)) * case["dim"] ** -0.5).masked_fill_(~_seen(case, q.device), -math.inf)


def _weights(state):
    case = state["case"]
    return state["lam"].expand(case["heads"]).view(case["kv_heads"], -1, 1, 1)


def _plain_diff(state):
    case = state["case"]
    B, S, H = case["batch"], case["seq"], case["heads"]
    s = _plain_scores(state)
    m = s.max(-1, keepdim=True).values
    e = s.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    lse = (m + total.log()).view(B, H, 2, S)
    maps = torch.matmul(e.div_(total), _values(state["v"], case, 1)[:, :, :, None])
    o = maps[:, :, :, 0] - _weights(state) * maps[:, :, :, 1]
    return _rows(o, case).to(BF16), _rows(maps[:, :, :, 1], case).to(BF16), lse


def _plain_diff_grad(state):
    case = state["case"]
    D, KH = case["dim"], case["kv_heads"]
    groups = case["heads"] // KH
    q, k = _split(state["q"], case, groups), _split(state["k"], case, 1)
    v, do = _values(state["v"], case, 1), _values(state["do"], case, groups)
    w = _weights(state)
    p = (_plain_scores(state) - state["lse"].view(case["batch"], KH, groups, 2, case["seq"], 1)).exp_()
    dv = torch.matmul((p[:, :, :, 0] - w * p[:, :, :, 1]).transpose(-1, -2), do).sum(2, keepdim=True)
    dp = torch.matmul(do, v.transpose(-1, -2))[:, :, :, None]
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p.mul_(dp - delta)
    ds[:, :, :, 1] *= -w
    dlam = -delta[:, :, :, 1, :, 0].sum((0, 3)).reshape(-1)
    dq = torch.matmul(ds, k) * D**-0.5
    dk = (torch.matmul(ds.transpose(-1, -2), q) * D**-0.5).sum(2, keepdim=True)
    return {"dq": _join(dq, case).to(BF16), "dk": _join(dk, case).to(BF16), "dv": _rows(dv, case).to(BF16), "dlam": dlam.sum().view(1) if case["shared"] else dlam}


# ----------------------------------------------------------------------------- one pass
def _scaling(case):
    from olmax_amd import ops

    return None if case["scaling"] == "none" else ops.RopeScaling(case["scaling"], case["factor"], original_length=case["original"])


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from olmax_amd import ops

        if kind == "tables":
            return ops.rotary_tables(case["length"], case["rotary"], state["theta"], "cuda", scaling=_scaling(case))
        if kind.startswith("rotate"):
            call = ops.rotary_fwd if kind == "rotate" else ops.rotary_bwd
            return call(state["x"], state["cos"], state["sin"], heads=case["heads"], head_dim=case["head_dim"], positions=state["positions"],
                        seq_len=case["seq"] or None, layout=case["layout"])
        kw = {"B": case["batch"], "S": case["seq"], "H": case["heads"], "KH": case["kv_heads"], "D": case["dim"], "window": case["window"] if case["window"] >= 0 else None}
        if kind == "diff":
            r = ops.diff_attn_fwd(state["q"], state["k"], state["v"], state["lam"], **kw)
            return {"o": r.o, "o2": r.o2, "lse": r.lse}
        dq, dk, dv, dlam = ops.diff_attn_bwd(state["q"], state["k"], state["v"], state["lam"], state["o"], state["o2"], state["lse"], state["do"], **kw)
        return {"dq": dq, "dk": dk, "dv": dv, "dlam": dlam}
    if kind == "tables":
        return _plain_tables(state["theta"], case, "cuda")
    if kind.startswith("rotate"):
        return _plain_rotate(state, 1.0 if kind == "rotate" else -1.0)
    if kind == "diff":
        o, o2, lse = _plain_diff(state)
        return {"o": o, "o2": o2, "lse": lse}
    return _plain_diff_grad(state)


# ----------------------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "tables":
        R, L, s, theta = case["rotary"], case["original"], case["factor"], state["theta"]
        freqs, size = [], 1.0
        for i in range(R // 2):
            f = math.exp(-2 * i / R * math.log(theta))
            if case["scaling"] == "linear":
                f /= s
            elif case["scaling"] == "llama3":
                wave = 2 * math.pi / f
                if wave > L:
                    f /= s
                elif wave >= L / 4:
                    part = (L / wave - 1) / 3
                    f = (1 - part) * f / s + part * f
            elif case["scaling"] == "yarn":
                lo = max(0, math.floor(R * math.log(L / (64 * math.pi), theta) / 2))
                hi = min(R - 1, math.ceil(R * math.log(L / (2 * math.pi), theta) / 2))
                part = min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))
                f = (1 - part) * f + part * f / s
                size = 1 + math.log(s) / 10
            freqs.append(f)
        angle = torch.outer(torch.arange(case["length"], dtype=F64, device="cuda"), torch.tensor(freqs, dtype=F64, device="cuda"))
        z = torch.polar(torch.full_like(angle, size), angle)
        return z.real.contiguous(), z.imag.contiguous()
    if case["kind"].startswith("rotate"):
        T, heads, D, R = case["tokens"], case["heads"], case["head_dim"], case["rotary"]
        x = state["x"].double().reshape(T, heads, D)
        p = _positions(state)
        z = torch.complex(state["cos"].double(), state["sin"].double())[p.clamp(min=0)]
        z = torch.where((p < 0)[:, None], torch.ones_like(z), z)[:, None]
        if case["kind"] == "rotate-grad":
            z = z.conj()
        turn = x[..., :R]
        pairs = turn.reshape(T, heads, 2, R // 2).transpose(-1, -2) if case["layout"] == "half" else turn.reshape(T, heads, R // 2, 2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        turn = (pairs.transpose(-1, -2) if case["layout"] == "half" else pairs).reshape(T, heads, R)
        return torch.cat([turn, x[..., R:]], -1).reshape(T, heads * D)
    # one sequence and head at a time; gradients of sum(o * do) by differentiation
    B, S, H, KH, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    grad = case["kind"] == "diff-grad"
    q, k, v = (state[n].double().view(B, S, -1, 2 * D) for n in "qkv")
    lam = state["lam"].double().expand(H)
    hidden = ~_seen(case, "cuda")
    outs = {n: torch.zeros_like(q) for n in (("dq",) if grad else ("o", "o2"))} | ({"dk": torch.zeros_like(k), "dv": torch.zeros_like(v)} if grad else {})
    lse, dlam = torch.zeros(B, H, 2, S, dtype=F64, device="cuda"), torch.zeros(H, dtype=F64, device="cuda")
    for b in range(B):
        for h in range(H):
            g = h // (H // KH)
            own_ = [t.clone().requires_grad_(grad) for t in (q[b, :, h], k[b, :, g], v[b, :, g], lam[h])]
            scores = [(own_[0][:, m * D: m * D + D] @ own_[1][:, m * D: m * D + D].T / math.sqrt(D)).masked_fill(hidden, -math.inf) for m in (0, 1)]
            second = torch.softmax(scores[1], 1) @ own_[2]
            o = torch.softmax(scores[0], 1) @ own_[2] - own_[3] * second
            if not grad:
                outs["o"][b, :, h], outs["o2"][b, :, h] = o, second
                lse[b, h, 0], lse[b, h, 1] = torch.logsumexp(scores[0], 1), torch.logsumexp(scores[1], 1)
                continue
            dq, dk, dv, dl = torch.autograd.grad(o, own_, state["do"].double().view(B, S, H, 2 * D)[b, :, h])
            outs["dq"][b, :, h] = dq
            outs["dk"][b, :, g] += dk
            outs["dv"][b, :, g] += dv
            dlam[h] += dl
    outs = {n: t.view(B * S, -1) for n, t in outs.items()}
    return outs | ({"dlam": dlam.sum().view(1) if case["shared"] else dlam} if grad else {"lse": lse})


def work(case):
    if case["kind"] == "tables":  # product, reduction and two polynomials of an angle
        n = case["length"] * (case["rotary"] // 2)
        return {"bytes": 8.0 * n, "flops": 40.0 * n}
    if case["kind"].startswith("rotate"):
        n = case["tokens"] * case["heads"]
        rows = min(case["tokens"], case["seq"] or case["tokens"])
        return {"bytes": 2.0 * n * case["head_dim"] * (4 if case["dtype"] == "f32" else 2) + 4.0 * rows * case["rotary"], "flops": 3.0 * n * case["rotary"]}
    B, S, H, KH, D, w = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim", "window"))
    w = S if w < 0 else min(w, S - 1)
    pairs = B * H * (S * (S + 1) / 2 - max(0, S - 1 - w) * (S - w) / 2)
    rows = 4.0 * B * S * D  # bytes of a row of 2D values in all places
    # both maps' scores, and one product of what they differ by with the values; five such products for the gradients
    if case["kind"] == "diff":
        return {"bytes": rows * (3 * H + 2 * KH) + 8.0 * B * S * H, "flops": 8.0 * D * pairs}
    return {"bytes": rows * (5 * H + 4 * KH) + 8.0 * B * S * H, "flops": 20.0 * D * pairs}
