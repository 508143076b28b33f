"""GPU parity tests of log probabilities, entropy, alternatives and distillation, on given logits and with the LM head, against the plain forms in 64 bits.

Tolerances count roundings of 2^-24 (u).  A score behind the row's largest, D = z - m, is a difference of logits times 1 / temperature (in
powers of two for an exponential): two roundings, and at most three of the factor, of which 2 u |D| are counted by themselves and 3 u |D| are within the 24 u below (|D| is 8 at
most where it has weight); a hardware exponential (2 u); a thread adds its share of the row one after another, V / (256 * 8 or 4) vectors behind an 8-fold
tree, and twelve more additions join the threads: CHAIN = V / 1024 + 24 u relative at most, for sums of positive numbers.
A soft-cap's tanh is off by 2^-22 at most (an exponential and a reciprocal, each halved by tanh's slope), its score by CAP = softcap * 2^-21 / temperature with its product's
rounding.  The temperature is the fp32 number that the kernel gets."""
import math

import numpy as np
import pytest
import torch

from oracle import ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def f32(x):
    return float(np.float32(x))


class Row:
    """What the bounds are made of, for each row of double logits."""

    def __init__(self, z, temperature=1.0, softcap=0.0):
        s = ref.token_scores(z, temperature, softcap)
        s = torch.where((s == -math.inf).all(1, keepdim=True), torch.zeros_like(s), s)
        self.D = s - s.max(1, keepdim=True).values
        self.p = torch.softmax(s, 1)
        lost = torch.where(self.p > 0, self.D, torch.zeros_like(self.D))
        self.first = (self.p * lost.abs()).sum(1)
        second = (self.p * lost ** 2).sum(1)
        self.lse = torch.logsumexp(self.D, 1)
        self.cap = softcap * 2.0 ** -21 / temperature
        self.chain = (z.shape[1] / 1024 + 24) * U
        # of ln S: the sum's relative error, the logarithm's own
        self.of_lse = self.chain + 2 * U * self.first + 3 * U * self.lse + 2 * U + 2 * self.cap
        self.of_entropy = (self.chain + self.cap) * (2 + 2 * self.first + self.lse) + 4 * U * second + 8 * U * (self.lse + self.first) + 4 * U

    def of_lp(self, lp):  # [T] or [T, k] log probabilities
        n = self.of_lse.view(-1, *[1] * (lp.dim() - 1))
        return n + self.cap + 3 * U * torch.nan_to_num(lp.abs(), posinf=0.0)


def near(got, want, bound, what):
    got = got.cpu().double()
    same = (got == want) | (got.isnan() & want.isnan())
    same |= got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound > torch.finfo(torch.float32).max)  # (fp32 has no such number)
    off = torch.where(same, torch.zeros_like(want), (got - want).abs() - bound)
    assert (off <= 0).all(), (what, got.flatten()[off.argmax()].item(), want.flatten()[off.argmax()].item(), off.max().item())


def check_scores(r, z, targets, top, temperature=1.0, softcap=0.0, rows=None):
    t = f32(temperature)
    lp, ent, best, ids = ref.token_logprobs_fwd(z, targets, top=top, temperature=t, softcap=f32(softcap))
    b = Row(z, t, f32(softcap))
    pick = (lambda x: x) if rows is None else (lambda x: x[rows])
    if targets is not None:
        near(pick(r.logprobs), lp, b.of_lp(lp), "logprobs")
    near(pick(r.entropy), ent, b.of_entropy, "entropy")
    if top:
        assert torch.equal(pick(r.top_ids).cpu().long(), ids)
        near(pick(r.top_logprobs), best, b.of_lp(best), "top_logprobs")
    return b


def make(T, V, dtype, seed=0, std=2.5):
    g = torch.Generator().manual_seed(seed * 1000 + V)
    z = torch.randn(T, V, generator=g) * std
    z[torch.arange(T), torch.randint(0, V, (T,), generator=g)] += torch.rand(T, generator=g) * 12
    targets = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    return z.to(dtype), targets


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 7, 9, 100, 1000, 4099, 16392, 50304, 100278])
@pytest.mark.parametrize("top,temperature,softcap", [(0, 1.0, 0.0), (5, 0.7, 0.0), (128, 1.0, 30.0)])
def test_scores(dtype, V, top, temperature, softcap):
    from olmax_amd import ops
    top = min(top, V)
    print(f"[case] score V{V} top{top}", flush=True)
    z, targets = make(7, V, dtype)
    targets[1], targets[2], targets[3] = -100, V, -5
    r = ops.token_logprobs(z.cuda(), targets.cuda(), top=top, temperature=temperature, softcap=softcap)
    check_scores(r, z.double(), targets, top, temperature, softcap)
    assert (r.stats[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,V,top", [(1100, 4099, 20), (1025, 1003, 128), (2100, 700, 0)])
def test_many_rows(dtype, T, V, top):
    """Rows that take a workgroup each."""
    from olmax_amd import ops
    z, targets = make(T, V, dtype)
    r = ops.token_logprobs(z.cuda(), targets.cuda(), top=top)
    check_scores(r, z.double(), targets, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [1001, 40005])
@pytest.mark.parametrize("T", [3, 1100])
def test_rows_anywhere(dtype, V, T):
    """Rows at any offset and stride, forward and backward, are the packed ones' bit for bit where both are cut alike, and within the bounds otherwise."""
    from olmax_amd import ops
    z, targets = make(T, V, dtype)
    wide = torch.full((T, V + 6), 99.0, dtype=dtype, device="cuda")
    wide[:, 5:5 + V] = z.cuda()
    view = wide[:, 5:5 + V]
    r = ops.token_logprobs(view, targets.cuda(), top=9)
    rows = torch.arange(min(T, 16)) if T < 20 else torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 555, T - 1])
    check_scores(r, z[rows].double(), targets[rows], 9, rows=rows)
    g = torch.randn(T, device="cuda")
    packed = ops.token_logprobs_bwd(z.cuda(), targets.cuda(), r.stats, g, dentropy=g)
    got = ops.token_logprobs_bwd(view, targets.cuda(), r.stats, g, dentropy=g)
    assert torch.equal(got, packed)  # (an element's gradient does not depend on who computes it)
    out = torch.full((T, V + 3), 7.0, dtype=dtype, device="cuda")
    ops.token_logprobs_bwd(view, targets.cuda(), r.stats, g, dentropy=g, out=out[:, 2:2 + V])
    assert torch.equal(out[:, 2:2 + V], packed) and (out[:, :2] == 7).all() and (out[:, 2 + V:] == 7).all()
    ops.token_logprobs_bwd(view, targets.cuda(), r.stats, g, dentropy=g, inplace=True)
    assert torch.equal(view, packed) and (wide[:, :5] == 99).all() and (wide[:, 5 + V:] == 99).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_gradients_between_the_logits(dtype):
    """Rows of logits and of their gradients that take turns in memory share none; gradients that overlap the logits are refused."""
    from olmax_amd import _lib, ops
    T, V = 5, 1003
    z, targets = make(T, V, dtype)
    both = torch.full((T, 2 * V), 5.0, dtype=dtype, device="cuda")
    both[:, :V] = z.cuda()
    r = ops.token_logprobs(both[:, :V], targets.cuda())
    g = torch.randn(T, device="cuda")
    ops.token_logprobs_bwd(both[:, :V], targets.cuda(), r.stats, g, out=both[:, V:])
    assert torch.equal(both[:, V:], ops.token_logprobs_bwd(z.cuda(), targets.cuda(), r.stats, g)) and torch.equal(both[:, :V].cpu(), z)
    with pytest.raises(_lib.OlmaxHipError, match="overlaps"):
        ops.token_logprobs_bwd(both[:, :V], targets.cuda(), r.stats, g, out=both[:, 1:V + 1])


def special(V, dtype):
    """Rows that masks and ties make; the targets name a token that has a probability where one has."""
    low = torch.finfo(dtype).min
    z, t = make(14, V, dtype, std=1.0)
    inf = math.inf
    z[0] = -inf                        # nothing left
    z[1] = low                         # the type's lowest value everywhere: a uniform row
    z[2] = -inf; z[2, V // 2] = 3.0    # one token left
    z[3] = -inf; z[3, V - 1] = 1.0; z[3, V // 3] = 1.0; z[3, 0] = 2.0
    z[4] = low; z[4, V - 2] = -5.0     # one above a mask of lowest values
    z[5] = 0.0                         # all the same
    z[6] = (torch.arange(V) % 3).to(dtype)  # a third of the row ties at the top
    z[7] = -1e6; z[7, 4] = -1e6 + 8192
    z[8] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(dtype)
    z[9] = 1000.0; z[9, 1::7] = 1004.0
    z[10, V // 2:] = -inf
    z[11, : V // 2] = low
    z[12] = torch.linspace(-20, 20, V).to(dtype)
    z[13] = torch.linspace(20, -20, V).to(dtype)
    t = torch.tensor([0, 3, V // 2, V // 3, V - 2, V - 1, 2, 4, 1, 1, 0, V - 1, V - 1, 0], dtype=torch.int32)
    return z, t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("temperature", [0.7, 3.0])
@pytest.mark.parametrize("V,copies", [(997, 1), (997, 80), (60001, 1), (60001, 40)])
def test_masks_and_ties_at_a_temperature(dtype, temperature, V, copies):
    """Scores beyond fp32 (the type's lowest value over 0.7) and far from 0: only differences of logits count."""
    from olmax_amd import ops
    print(f"[case] special V{V} x{copies} temperature {temperature}", flush=True)
    z, t = special(V, dtype)
    z[12], z[13] = 1e30, -3e38
    z[13, 5] = torch.finfo(dtype).max / 2
    t[12], t[13] = 7, 5
    r = ops.token_logprobs(z.repeat(copies, 1).cuda(), t.repeat(copies).cuda(), top=20, temperature=temperature)
    for c in range(min(copies, 4)):
        check_scores(r, z.double(), t, 20, temperature, rows=torch.arange(14) + 14 * c)
    k = 8
    ids = torch.stack([(t.long() + 3 * j) % V for j in range(k)], 1).to(torch.int32)  # the first has a probability where one has
    q = torch.full((14, k), -math.inf)
    q[:, 0] = -0.25                                                                  # (what a student rules out costs infinitely much)
    ids, q = ids[1:], q[1:]                                                          # (a row of nothing has no distribution)
    for tail in ("renormalize", "bucket"):
        rows = list(range(13)) if tail == "renormalize" else [0, 4, 5, 7, 8, 9, 10, 11]  # (nor do the others of rows of one token)
        per, bound, grad, gbound = distill_bounds(z[1:][rows], ids[rows], q[rows], tail, temperature, 0.0, torch.ones(len(rows)))
        n = len(rows)
        loss, d = ops.distill(z[1:][rows].repeat(copies, 1).cuda(), ids[rows].repeat(copies, 1).cuda(), q[rows].repeat(copies, 1).cuda(), tail=tail, temperature=temperature,
                              reduction="none")
        for c in range(min(copies, 4)):
            near(loss[n * c:n * c + n], per, bound, tail)
            near(d[n * c:n * c + n], grad, gbound, tail)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V,copies", [(997, 1), (997, 100), (60001, 1), (60001, 80)])
@pytest.mark.parametrize("top", [1, 20, 128])
def test_masks_and_ties(dtype, V, copies, top):
    """Few rows, in parts, and many whole ones.  Among equal logits the lowest index, behind all of them the masked tokens by index."""
    from olmax_amd import ops
    print(f"[case] special V{V} x{copies} top{top}", flush=True)
    z, t = special(V, dtype)
    r = ops.token_logprobs(z.repeat(copies, 1).cuda(), t.repeat(copies).cuda(), top=top)
    # A copy begins 14 V elements on, a multiple of 4 bytes: rows of other copies are cut into vectors elsewhere and their sums are grouped otherwise, but four copies are
    # a multiple of 16 bytes, so every fourth is the first bit for bit.
    for c in range(min(copies, 4)):
        check_scores(r, z.double(), t, top, rows=torch.arange(14) + 14 * c)
    for a in r:
        a = a.view(copies, -1)[::4]
        assert ((a == a[:1]) | (a.isnan() & a[:1].isnan())).all()
    assert torch.equal(r.top_ids.view(copies, -1), r.top_ids.view(copies, -1)[:1].expand(copies, -1))
    g = torch.linspace(-1, 1, 14)
    got = ops.token_logprobs_bwd(z.cuda(), t.cuda(), r.stats[:14].contiguous(), g.cuda(), dentropy=g.flip(0).contiguous().cuda())
    want, bound = score_grads(z, t, g, g.flip(0))
    near(got, want, bound, "dlogits")


def score_grads(z, t, g, h, temperature=1.0, softcap=0.0):
    """The exact gradient and its bound: p is off by the bounds of its logarithm, the bracket by those of entropy and logarithm, the soft-cap's slope 1 - tanh^2 by 2^-20;
    a target adds its cotangent; then one rounding to the type."""
    tau, cap = f32(temperature), f32(softcap)
    zd, gd = z.double(), g.double()
    hd = torch.zeros_like(gd) if h is None else h.double()
    want = ref.token_logprobs_bwd(zd, t, gd, None if h is None else hd, temperature=tau, softcap=cap)
    b = Row(zd, tau, cap)
    logp = torch.where(b.p > 0, b.p.log(), torch.zeros_like(b.p))
    lp = (b.of_lse + b.cap)[:, None] + 3 * U * (logp.abs() + b.D.clamp(min=-200).abs())
    inner = gd.abs()[:, None] + hd.abs()[:, None] * (logp.abs() + (b.lse + b.first)[:, None])
    raw = b.p * (inner * (lp + 8 * U) + hd.abs()[:, None] * (lp + b.of_entropy[:, None])) / tau
    hit = torch.zeros_like(b.p).scatter(1, t.clamp(0, z.shape[1] - 1).long()[:, None], gd.abs()[:, None]) * 4 * U / tau
    slope = 2.0 ** -20 * (b.p * inner + hit / (4 * U)) / tau if softcap else 0.0
    # half a step of the type; below its normal range a step is 2^-133 (bf16) or 2^-149, and an exponential below 2^-126 may be flushed
    return want, raw + hit + slope + torch.finfo(z.dtype).eps / 2 * want.abs() * (1 + 2 ** -10) + 2.0 ** -120


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 9, 1000, 4099, 50304, 100278])
@pytest.mark.parametrize("temperature,softcap,entropy", [(1.0, 0.0, True), (0.7, 0.0, False), (2.0, 30.0, True)])
def test_score_gradients(dtype, V, temperature, softcap, entropy):
    from olmax_amd import ops
    print(f"[case] score grad V{V}", flush=True)
    z, t = make(6, V, dtype)
    t[1], t[2] = -100, V
    g = torch.tensor([1.0, 5.0, -3.0, -0.5, 0.0, 2.0])
    h = torch.tensor([0.1, 7.0, 0.3, -0.2, 1.0, 0.0]) if entropy else None
    kw = dict(temperature=temperature, softcap=softcap)
    r = ops.token_logprobs(z.cuda(), t.cuda(), **kw)
    got = ops.token_logprobs_bwd(z.cuda(), t.cuda(), r.stats, g.cuda(), dentropy=None if h is None else h.cuda(), **kw)
    want, bound = score_grads(z, t, g, h, temperature, softcap)
    near(got, want, bound, "dlogits")
    assert (got[1] == 0).all()


def test_not_a_number_stays_in_its_row():
    from olmax_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        for V in (300, 50001):
            z, t = make(5, V, dtype)
            z[1, 7] = math.nan
            z[3, 9] = math.inf
            z[4, V - 1] = math.nan
            for x in (z, z.repeat(300, 1)):
                r = ops.token_logprobs(x.cuda(), t.repeat(x.shape[0] // 5).cuda(), top=20)
                bad = torch.tensor([False, True, False, True, True]).repeat(x.shape[0] // 5)
                assert r.entropy.isnan().cpu().equal(bad) and r.logprobs.isnan().cpu().equal(bad)
                ids = r.top_ids.cpu().long()
                assert ((ids >= 0) & (ids < V)).all() and all(len(set(i.tolist())) == 20 for i in ids[:5])
                check_scores(r, z[[0, 2]].double(), t[[0, 2]], 20, rows=torch.tensor([0, 2]))


def test_no_targets_and_outputs_that_are_not_asked_for():
    from olmax_amd import ops
    z, t = make(4, 3001, torch.float32)
    a, b = ops.token_logprobs(z.cuda(), top=3), ops.token_logprobs(z.cuda(), t.cuda())
    assert a.logprobs is None and b.top_ids is None and torch.equal(a.entropy, b.entropy) and torch.equal(a.stats, b.stats)
    check_scores(a, z.double(), None, 3)


# ----------------------------------------------------------------------------- distillation
def teacher(z, k, seed=1):
    g = torch.Generator().manual_seed(seed)
    u = z.double() * 0.8 + torch.randn(z.shape, generator=g, dtype=torch.float64)
    t, ids = torch.topk(torch.log_softmax(u, 1), k, dim=1)
    return ids.to(torch.int32), t.float()


def distill_bounds(z, ids, t, tail, temperature, softcap, dl):
    """(row loss, its bound, gradient, its bound); dl: what each row's gradient is scaled by."""
    tau, cap = f32(temperature), f32(softcap)
    zd, td = z.double(), t.double()
    kw = dict(tail=tail, temperature=tau, softcap=cap, reduction="none")
    per = ref.distill_fwd(zd, ids, td, **kw)
    grad = ref.distill_bwd(zd, ids, td, dloss=dl.double(), **kw)
    b = Row(zd, tau, cap)
    V = z.shape[1]
    q, logq, r, ok = ref._teacher(ids.long(), td, V, tail, tau)
    logp = ref._log_softmax(ref.token_scores(zd, tau, cap))
    lp = logp.gather(1, ids.long().clamp(0, V - 1))
    lq = torch.where(q > 0, logq, torch.zeros_like(q))
    lp = torch.where(q > 0, lp, torch.zeros_like(q))
    k = ids.shape[1]
    # q: exponentials of arguments up to |ln q| (and t's range / tau), a sum of k of them; r is 1 minus that
    of_q = q * (4 * U * lq.abs() + 8 * U) + q * 8 * U
    of_r = of_q.sum(1) + 10 * U
    terms = (of_q * (lq - lp).abs() + q * (b.of_lp(lp) + 8 * U * (lq.abs() + lp.abs()) + 12 * U)).sum(1) + k * U * (q * (lq - lp).abs()).sum(1)
    bound = terms + 4 * U * per.abs() + 4 * U
    a = torch.ones_like(r)
    of_a = of_r + 4 * U
    if tail == "bucket":
        hidden = torch.zeros(z.shape[0], V + 1, dtype=torch.bool).scatter(1, torch.where(ok, ids.long(), V), True)[:, :V]
        s = torch.where(hidden, 0.0, b.p).sum(1)
        ratio = torch.where(r > 0, r / s, torch.zeros_like(r))
        log_ratio = torch.where(r > 0, ratio.log().abs() + r.log().abs() + s.log().abs(), torch.zeros_like(r))
        other = b.of_lse + b.chain + 2 * U * (b.p * torch.where(hidden, 0.0, b.D).abs()).nan_to_num().sum(1) / s.clamp(min=1e-300) + 4 * U
        bound = bound + of_r * (log_ratio + 1) + r * (other + 6 * U * log_ratio) + 2 * U
        a = 1 - ratio
        of_a = of_r + of_r / s.clamp(min=1e-300) + ratio * (other + 6 * U) + 4 * U
    wide = b.p * ((b.of_lse + b.cap)[:, None] + 4 * U * b.D.clamp(min=-200).abs() + 12 * U)
    raw = wide * torch.maximum(a.abs(), torch.ones_like(a))[:, None] + b.p * of_a[:, None]
    raw = raw.scatter_add(1, ids.long().clamp(0, V - 1), of_q + 4 * U * q)
    if softcap:
        raw = raw + 2.0 ** -20 * torch.maximum(grad.abs() * tau / dl.double().abs().clamp(min=1e-300)[:, None], b.p + torch.zeros_like(b.p).scatter_add(1, ids.long().clamp(0, V - 1), q))
    gbound = raw * dl.double().abs()[:, None] / tau + torch.finfo(z.dtype).eps / 2 * (1 + 2 ** -10) * grad.abs() + 2.0 ** -120
    return per, bound, grad, gbound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 9, 1000, 4099, 16400, 50304, 100278])
@pytest.mark.parametrize("k", [1, 7, 128])
@pytest.mark.parametrize("tail,temperature,softcap", [("renormalize", 1.0, 0.0), ("renormalize", 2.0, 30.0), ("bucket", 1.0, 0.0), ("bucket", 0.7, 30.0)])
def test_distill(dtype, V, k, tail, temperature, softcap):
    from olmax_amd import ops
    k = min(k, V)
    print(f"[case] distill V{V} k{k} {tail}", flush=True)
    z, _ = make(5, V, dtype)
    ids, t = teacher(z, k)
    dl = torch.tensor([1.0, -2.0, 0.5, 3.0, 1.0])
    if V > 9 and k > 5:
        ids[1, 3] = ids[1, 0]    # named again
        ids[2, 1], ids[2, 2] = -1, V
        t[3, 2] = -math.inf      # the teacher rules it out
    ids[4, 0] = -3               # left out
    per, bound, grad, gbound = distill_bounds(z, ids, t, tail, temperature, softcap, dl)
    kw = dict(tail=tail, temperature=temperature, softcap=softcap)
    loss, d = ops.distill(z.cuda(), ids.cuda(), t.cuda(), reduction="none", dloss_rows=dl.cuda(), **kw)
    near(loss, per, bound, "row losses")
    near(d, grad, gbound, "dlogits")
    assert (d[4] == 0).all() and loss[4] == 0
    alone, none = ops.distill(z.cuda(), ids.cuda(), t.cuda(), reduction="none", want_grad=False, **kw)
    assert none is None and torch.allclose(alone, loss, rtol=2e-6, atol=2e-6)
    mean, dm = ops.distill(z.cuda(), ids.cuda(), t.cuda(), dloss=2.0, **kw)
    assert abs(mean.item() - per[:4].mean().item()) <= bound[:4].mean().item() + 4 * U * per[:4].abs().mean().item()
    near(dm, *distill_bounds(z, ids, t, tail, temperature, softcap, torch.full((5,), 0.5))[2:], "mean's dlogits")
    total, _ = ops.distill(z.cuda(), ids.cuda(), t.cuda(), reduction="sum", inplace=False, **kw)
    assert abs(total.item() - per.sum().item()) <= bound.sum().item() + 8 * U * per.abs().sum().item()
    wide = torch.full((5, V + 5), 9.0, dtype=dtype, device="cuda")
    wide[:, 3:3 + V] = z.cuda()
    ops.distill(wide[:, 3:3 + V], ids.cuda(), t.cuda(), dloss=2.0, inplace=True, **kw)
    near(wide[:, 3:3 + V], *distill_bounds(z, ids, t, tail, temperature, softcap, torch.full((5,), 0.5))[2:], "in place, elsewhere")
    assert (wide[:, :3] == 9).all() and (wide[:, 3 + V:] == 9).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,V", [(1, 102401), (40, 262147), (200, 16386), (200, 102408), (200, 163841), (130, 262147), (405, 50304), (405, 102408), (405, 163848), (260, 1000003)])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_distill_rows_held_and_in_shares(dtype, T, V, tail):
    """Lengths about those that 256, 512 and 1024 threads hold, of few rows and of many, with the gradient and without."""
    from olmax_amd import ops
    print(f"[case] distill T{T} V{V} {tail}", flush=True)
    z, _ = make(3, V, dtype)
    ids, t = teacher(z, 33)
    ids[0, 4], ids[1, 5] = V - 1, 0  # the row's ends
    per, bound, grad, gbound = distill_bounds(z, ids, t, tail, 1.0, 0.0, torch.ones(3))
    n = (T + 2) // 3
    rows, ids, t = z.cuda().repeat(n, 1)[:T], ids.cuda().repeat(n, 1)[:T], t.cuda().repeat(n, 1)[:T]
    loss, d = ops.distill(rows, ids, t, tail=tail, reduction="none")
    alone, _ = ops.distill(rows, ids, t, tail=tail, reduction="none", want_grad=False)
    for i in range(0, T, 1 if T < 50 else 37):
        for got in (loss, alone):
            near(got[i:i + 1], per[i % 3:i % 3 + 1], bound[i % 3:i % 3 + 1], f"row loss {i}")
        near(d[i], grad[i % 3], gbound[i % 3], f"dlogits {i}")
    mean, dmean = ops.distill(rows, ids, t, tail=tail, inplace=True)
    assert dmean.data_ptr() == rows.data_ptr()
    want = per[torch.arange(T) % 3]
    near(mean, want.mean(), bound[torch.arange(T) % 3].mean() + (T / 1024 + 12) * U * want.abs().mean(), "mean")
    for i in (0, T // 2, T - 1):
        near(dmean[i], grad[i % 3] / T, gbound[i % 3] / T + 3 * U * grad[i % 3].abs() / T + 2.0 ** -120, f"dlogits of the mean {i}")


def test_offsets_beyond_32_bits():
    """Rows of 4.4 G logits: the last ones are the first bit for bit, forward and, in place, backward."""
    from olmax_amd import ops
    T, V = 22000, 200000
    z, targets = make(8, V, torch.bfloat16)
    ids, t = teacher(z, 16)
    few = z.cuda()
    targets, ids, t, g = targets.cuda(), ids.cuda(), t.cuda(), torch.randn(8, device="cuda")
    many = few.repeat(T // 8, 1)
    large = lambda x: x.repeat(T // 8, *[1] * (x.dim() - 1))  # noqa: E731
    r = ops.token_logprobs(many, large(targets), top=5)
    check_scores(r, z.double(), targets.cpu(), 5, rows=torch.arange(T - 8, T))
    for a in r:
        assert torch.equal(a[:8], a[T - 8:])
    loss, d = ops.distill(many, large(ids), large(t), tail="bucket", reduction="none")
    assert torch.equal(loss[:8], loss[T - 8:]) and torch.equal(d[:8], d[T - 8:]) and torch.equal(d[:8], d[T // 2:T // 2 + 8])
    del d
    ops.token_logprobs_bwd(many, large(targets), r.stats, large(g), inplace=True)
    want = ops.token_logprobs_bwd(few, targets, r.stats[:8].contiguous(), g)
    assert torch.equal(many[:8], want) and torch.equal(many[T - 8:], want)


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_distill_many_rows(tail):
    """More rows than a workgroup counts by itself, some left out."""
    from olmax_amd import ops
    z, _ = make(2500, 801, torch.bfloat16)
    ids, t = teacher(z, 10)
    ids[5::9, 0] = -1
    kept = int((ids[:, 0] >= 0).sum())
    loss, d = ops.distill(z.cuda(), ids.cuda(), t.cuda(), tail=tail)
    per, bound, grad, gbound = distill_bounds(z, ids, t, tail, 1.0, 0.0, torch.full((2500,), 1.0 / kept))
    assert abs(loss.item() - per.sum().item() / kept) <= bound.sum().item() / kept + 16 * U * per.abs().sum().item() / kept
    near(d, grad, gbound, "dlogits")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_distill_rows_of_masks(dtype, tail):
    from olmax_amd import ops
    V, k = 5003, 6
    z, _ = special(V, dtype)
    ids = torch.stack([torch.randperm(V, generator=torch.Generator().manual_seed(i))[:k] for i in range(14)]).to(torch.int32)
    ids[2, 0], ids[3, :3] = V // 2, torch.tensor([0, V - 1, V // 3])
    t = torch.log_softmax(torch.randn(14, k, generator=torch.Generator().manual_seed(9)), 1) - 0.3
    # rows whose teacher names masked tokens have an infinite loss (2, 3, 4 and 7 keep a finite gradient)
    for x in (z, ):
        loss, d = ops.distill(x.cuda(), ids.cuda(), t.cuda(), tail=tail, reduction="none")
        assert loss[0] == 0 and (d[0] == 0).all()
        per, bound, grad, gbound = distill_bounds(z, ids, t, tail, 1.0, 0.0, torch.ones(14))
        fine = [1, 5, 6, 8, 9, 12, 13]
        near(loss[fine], per[fine], bound[fine], "row losses")
        near(d[fine], grad[fine], gbound[fine], "dlogits")
        assert loss[2] == math.inf and torch.isfinite(d).all()


def test_distilling_a_distribution_into_itself_is_nothing():
    """The teacher's pass of the same logits: the loss and the gradient vanish but for the roundings of q and p, 2^-19 each over 8 tokens and a row's sum."""
    from olmax_amd import ops
    z, _ = make(40, 5000, torch.float32)
    r = ops.token_logprobs(z.cuda(), top=8)
    loss, d = ops.distill(z.cuda(), r.top_ids, r.top_logprobs, tail="bucket", reduction="none")
    assert loss.abs().max() < 2 ** -18 and d.abs().max() < 2 ** -18


# ----------------------------------------------------------------------------- with the LM head
def head(T, d, V, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(T, d, device="cuda", generator=g).bfloat16()
    W = (torch.randn(V, d, device="cuda", generator=g) * 2 / math.sqrt(d)).bfloat16()
    t = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    return h, W, t


HEADS = [(1, 64, 100), (5, 256, 4096), (33, 100, 777), (37, 200, 1003), (300, 320, 1030), (513, 1024, 5000), (1024, 512, 2304), (700, 72, 50304),
         (33, 1032, 8001), (63, 2048, 4001)]  # (gradients of 64 tokens)
# large tiles, the logits in the accumulators: whole rounds of tiles and columns behind them; partial tiles and k-tiles; a row length that is no multiple of 8, with and without
# columns behind the last round; one round exactly
IN_TILES = [(256, 64, 70000), (511, 72, 40007), (700, 128, 50301), (512, 256, 32768)]
# fewer tokens than a tile has rows, padded: fewer than a k-tile of dW has, one more than the logits are padded from, a row length that is no multiple of 8
PADDED = [(5, 64, 70000), (40, 128, 50301), (64, 64, 70001), (65, 72, 70000), (130, 256, 40007), (255, 64, 70000)]


@pytest.mark.parametrize("T,d,V", IN_TILES + PADDED)
@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (0.7, 20.0)])
def test_lmhead_in_tiles(T, d, V, temperature, softcap):
    """The bounds of the two tests below, on the GPU in 64 bits; targets in every 256 columns, some ignored, some out of range, no cotangent of the entropy."""
    from olmax_amd import ops
    print(f"[case] tiles {T} {d} {V}", flush=True)
    if T > 64:
        assert ops._size("olmax_lmhead_logprobs_workspace_bytes", T, d, V, 0) < 2 * T * V  # (fp32 logits would need 4)
    if T < 256:
        assert ops._size("olmax_lmhead_logprobs_bwd_workspace_bytes", T, d, V) > 2 * 256 * V
    h, W, t = head(T, d, V)
    t = ((torch.arange(T, device="cuda") * 977 + 255) % V).to(torch.int32)
    t[0], t[1], t[2], t[3], t[4], t[T - 1] = V - 1, -100, V, -7, 0, V - 2
    tau, cap = f32(temperature), f32(softcap)
    r = ops.lmhead_logprobs(h, W, t, temperature=temperature, softcap=softcap)
    z = h.double() @ W.double().t()
    of_z = (4 * math.sqrt(d) * U * (h.double().abs() @ W.double().abs().t()).max(1).values).cpu() / tau
    s = ref.token_scores(z, tau, cap)
    logp = torch.log_softmax(s, 1)
    p = logp.exp()
    entropy = -(p * logp).sum(1)
    inside = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1).long()[:, None]
    lp = torch.where(inside, logp.gather(1, at)[:, 0], 0.0)
    kept = t != -100
    b = Row(z[:300].cpu(), tau, cap)
    few = slice(0, b.lse.shape[0])
    near(r.logprobs[few], (lp * kept)[few].cpu(), b.of_lp((lp * kept)[few].cpu()) + 2 * of_z[few], "logprobs")
    near(r.entropy[few], (entropy * kept)[few].cpu(), b.of_entropy + 2 * of_z[few] * (1 + b.first + b.lse), "entropy")
    near(r.logprobs, (lp * kept).cpu(), b.of_lp((lp * kept)[few].cpu()).max() + 2 * of_z, "logprobs of all rows, the largest bound of some")
    assert torch.equal((r.stats[:, 2]), r.entropy) and (r.stats[1] == 0).all()
    g = torch.randn(T, device="cuda")
    dh, dW = ops.lmhead_logprobs_bwd(h, W, t, r.stats, g, temperature=temperature, softcap=softcap)
    gd = (g.double() * inside * kept)[:, None]
    dz = (-gd * p).scatter_add(1, at, gd) / tau
    if softcap:
        dz = dz * (1 - torch.tanh(z / cap) ** 2)
    for got, want in ((dh, dz @ W.double()), (dW, dz.t() @ h.double())):
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()
        assert (got[-40:].double() - want[-40:]).norm() <= 2.0 ** -7 * want[-40:].norm()
    assert (dh[1:4] == 0).all()


@pytest.mark.parametrize("T,d,V", HEADS)
@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (0.7, 20.0)])
def test_lmhead_scores(T, d, V, temperature, softcap):
    """A logit is a sum of d exact products in fp32, at most d additions behind one another and as many in the matrix instructions: off by d u sum |h w| at worst, and as
    roundings are as often up as down, by some sqrt(d); the bound takes 4 sqrt(d) u sum |h w|, |h| |W^T| at its largest in the row."""
    from olmax_amd import ops
    print(f"[case] lmhead {T} {d} {V}", flush=True)
    h, W, t = head(T, d, V)
    if T > 4:
        t[3] = -100
    r = ops.lmhead_logprobs(h, W, t, temperature=temperature, softcap=softcap)
    with_top = ops.lmhead_logprobs(h, W, t, top=min(V, 10), temperature=temperature, softcap=softcap)
    z = (h.double() @ W.double().t()).cpu()
    of_z = (4 * math.sqrt(d) * U * (h.double().abs() @ W.double().abs().t()).max(1).values).cpu() / f32(temperature)
    lp, ent, best, ids = ref.token_logprobs_fwd(z, t.cpu(), top=min(V, 10), temperature=f32(temperature), softcap=f32(softcap))
    b = Row(z, f32(temperature), f32(softcap))
    for x in (r, with_top):
        near(x.logprobs, lp, b.of_lp(lp) + 2 * of_z, "logprobs")
        near(x.entropy, ent, b.of_entropy + 2 * of_z * (1 + b.first + b.lse), "entropy")
    near(with_top.top_logprobs, best, b.of_lp(best) + 2 * of_z[:, None], "top_logprobs")  # (the ids where two logits are that near may change places)
    kept = ids[:, 0] >= 0
    near(z[kept].gather(1, with_top.top_ids.cpu().long()[kept]), z[kept].gather(1, ids[kept]), 2 * of_z[kept][:, None] * f32(temperature), "top_ids")


def product_bound(d, want, T):
    """dlogits rounded to bf16 (2^-9 rms of itself), fp32 sums, the result to bf16 (2^-8 at most): in the norm 2^-8 of both together."""
    return 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("T,d,V", HEADS)
@pytest.mark.parametrize("temperature,softcap,dw_f32", [(1.0, 0.0, False), (0.7, 20.0, True)])
def test_lmhead_score_gradients(T, d, V, temperature, softcap, dw_f32):
    from olmax_amd import ops
    print(f"[case] lmhead grad {T} {d} {V}", flush=True)
    h, W, t = head(T, d, V)
    if T > 4:
        t[3] = -100
    g, e = torch.randn(T, device="cuda"), torch.randn(T, device="cuda") * 0.3
    kw = dict(temperature=temperature, softcap=softcap)
    stats = ops.lmhead_logprobs(h, W, t, **kw).stats
    dh, dW = ops.lmhead_logprobs_bwd(h, W, t, stats, g, dentropy=e, dw_f32=dw_f32, **kw)
    z = (h.double() @ W.double().t()).cpu()
    dz = ref.token_logprobs_bwd(z, t.cpu(), g.cpu().double(), e.cpu().double(), temperature=f32(temperature), softcap=f32(softcap)).cuda()
    assert dW.dtype == (torch.float32 if dw_f32 else torch.bfloat16)
    for got, want in ((dh, dz @ W.double()), (dW, dz.t() @ h.double())):
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()
    only, none = ops.lmhead_logprobs_bwd(h, W, t, stats, g, dentropy=e, want_dw=False, **kw)
    assert none is None and (only.double() - dh.double()).norm() <= 2.0 ** -8 * dh.double().norm()
    none, only = ops.lmhead_logprobs_bwd(h, W, t, stats, g, dentropy=e, want_dh=False, **kw)
    assert none is None and (only.double() - dW.double()).norm() <= 2.0 ** -8 * dW.double().norm()


@pytest.mark.parametrize("T,d,V", HEADS + PADDED)
@pytest.mark.parametrize("tail,temperature,softcap", [("renormalize", 2.0, 0.0), ("bucket", 1.0, 20.0)])
def test_lmhead_distill(T, d, V, tail, temperature, softcap):
    from olmax_amd import ops
    h, W, _ = head(T, d, V)
    z = (h.double() @ W.double().t()).cpu()
    ids, t = teacher(z, 9)
    if T > 4:
        ids[2, 0] = -1
    loss, dh, dW = ops.lmhead_distill(h, W, ids.cuda(), t.cuda(), tail=tail, temperature=temperature, softcap=softcap, dloss=3.0)
    kw = dict(tail=tail, temperature=f32(temperature), softcap=f32(softcap))
    dz = ref.distill_bwd(z, ids, t.double(), dloss=3.0, **kw).cuda()
    want = ref.distill_fwd(z, ids, t.double(), **kw)
    of_z = 4 * math.sqrt(d) * U * (h.double().abs() @ W.double().abs().t()).max().item()
    assert abs(loss.item() - want.item()) <= 3 * of_z + 2.0 ** -19 * (1 + abs(want.item()))
    for got, w in ((dh, dz @ W.double()), (dW, dz.t() @ h.double())):
        assert (got.double() - w).norm() <= 2.0 ** -8 * w.norm()
    alone = ops.lmhead_distill(h, W, ids.cuda(), t.cuda(), tail=tail, temperature=temperature, softcap=softcap, want_dh=False, want_dw=False)
    assert alone[1] is None and alone[2] is None and abs(alone[0].item() - loss.item()) <= 2.0 ** -20 * (1 + abs(loss.item()))


# ----------------------------------------------------------------------------- together, as they are used
def test_a_teacher_a_student_and_a_policy_step():
    """A teacher's pass, a student's distillation from what it wrote (padded rows and all), and a policy-gradient step on the student's tokens, on a stream of its own."""
    from olmax_amd import ops
    T, d, V = 257, 256, 3000
    ht, Wt, targets = head(T, d, V, 1)
    hs, Ws, _ = head(T, d, V, 2)
    targets[200:] = -100  # padding
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        notes = ops.lmhead_logprobs(ht, Wt, targets, top=16)
        loss, dh, dW = ops.lmhead_distill(hs, Ws, notes.top_ids, notes.top_logprobs, tail="bucket")
        now = ops.lmhead_logprobs(hs, Ws, targets)
        ratio_grad = -torch.exp(now.logprobs - now.logprobs.detach())
        ph, pW = ops.lmhead_logprobs_bwd(hs, Ws, targets, now.stats, ratio_grad, dentropy=torch.full_like(ratio_grad, -0.01))
    torch.cuda.current_stream().wait_stream(s)
    assert (notes.top_ids[200:] == -1).all() and (dh[200:] == 0).all() and (ph[200:] == 0).all()
    z = (hs.double() @ Ws.double().t()).cpu()
    ids, t = notes.top_ids.cpu(), notes.top_logprobs.cpu().double()
    want = ref.distill_fwd(z, ids, t, tail="bucket")
    assert abs(loss.item() - want.item()) <= 2.0 ** -17 * (1 + want.item())
    dz = ref.distill_bwd(z, ids, t, tail="bucket").cuda()
    pz = ref.token_logprobs_bwd(z, targets.cpu(), ratio_grad.cpu().double(), torch.full((T,), -0.01, dtype=torch.float64)).cuda()
    for got, w in ((dh, dz @ Ws.double()), (dW, dz.t() @ hs.double()), (ph, pz @ Ws.double()), (pW, pz.t() @ hs.double())):
        assert (got.double() - w).norm() <= 2.0 ** -8 * w.norm()


@pytest.mark.parametrize("T,V", [(3, 40000), (1100, 900)])
def test_recorded_calls_replay(T, V):
    """All row operators in one graph, replayed four times over changing logits with eager work in between; results are bit-equal to the eager ones."""
    from olmax_amd import ops
    make_z = lambda i: make(T, V, torch.bfloat16, seed=i)[0].cuda()  # noqa: E731
    z, t = make_z(0), make(T, V, torch.bfloat16)[1].cuda()
    g = torch.randn(T, device="cuda")

    def work():
        r = ops.token_logprobs(z, t, top=12)
        d = ops.token_logprobs_bwd(z, t, r.stats, g, dentropy=g)
        loss, dd = ops.distill(z, r.top_ids, r.top_logprobs, tail="bucket", temperature=1.5)
        return [*r, d, loss, dd]
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        z.copy_(make_z(i + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


def test_results_repeat():
    from olmax_amd import ops
    z, t = special(60001, torch.bfloat16)
    z, t = z.cuda(), t.cuda()
    first = ops.token_logprobs(z, t, top=128)
    for _ in range(5):
        again = ops.token_logprobs(z, t, top=128)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def _all_calls(T, V, d, seed):
    """Every row operator and every form with the LM head, on inputs of their own: a call that returns all results."""
    from olmax_amd import ops
    z, t = make(T, V, torch.bfloat16, seed=seed)
    g = torch.Generator().manual_seed(seed)
    h, W = (torch.randn(n, d, generator=g).to(torch.bfloat16).cuda() for n in (T, V))
    z, t, c = z.cuda(), t.cuda(), torch.randn(T, generator=g).cuda()

    def work():
        r = ops.token_logprobs(z, t, top=12)
        s = ops.lmhead_logprobs(h, W, t, temperature=8.0)
        return [*r, ops.token_logprobs_bwd(z, t, r.stats, c, dentropy=c), *ops.distill(z, r.top_ids, r.top_logprobs, tail="bucket"), s.logprobs, s.entropy, s.stats,
                *ops.lmhead_logprobs_bwd(h, W, t, s.stats, c, temperature=8.0), *ops.lmhead_distill(h, W, r.top_ids, r.top_logprobs, temperature=8.0)]
    return work


def test_two_streams_at_once():
    """Calls on two streams whose work overlaps, with workspaces from one allocator, leave the results of calls by themselves."""
    works = [_all_calls(5, 40000, 64, 1), _all_calls(300, 9001, 128, 2)]
    want = [[x.clone() for x in w()] for w in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    got = [[], []]
    for _ in range(6):
        for i, (s, w) in enumerate(zip(streams, works)):
            with torch.cuda.stream(s):
                got[i].append(w())
    torch.cuda.synchronize()
    for many, one in zip(got, want):
        for results in many:
            assert all(torch.equal(a, b) for a, b in zip(results, one))


def test_two_graphs_that_share_their_memory():
    """Graphs recorded into one pool, whose workspaces may lie in the same place, replayed in turn: each leaves its own results."""
    works = [_all_calls(5, 40000, 64, 1), _all_calls(300, 9001, 128, 2)]
    want = [[x.clone() for x in w()] for w in works]
    torch.cuda.synchronize()
    pool, graphs, outs = None, [], []
    for w in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(w())
        pool = graph.pool()
        graphs.append(graph)
    for i in (0, 1, 1, 0, 1, 0):
        graphs[i].replay()
        works[1 - i]()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
