"""The bucket of all other tokens in a distillation, where the teacher's tokens lead by so much that the probability of the others leaves fp32.

With m' the others' largest score and S' = sum exp(z - m') over them, ln s = (m' - m) + ln S' - ln S and the others' gradient is p_i (sum q + r) - r exp(z_i - m') / S'.  The tolerances
count roundings of u = 2^-24.  A difference of scores, D, is off by 5 u |D| (two roundings and three of the factor), a soft-capped score by cap = softcap * 2^-21 / temperature.  S' may be
taken against a score that is up to 47 above m' (where a row is held in registers), and is off by a sum's chain, V / 1024 + 24 u, and by what its terms' differences are; the exponential and the
logarithm are off by 2 u, and what is added up to a logarithm by 3 u of itself."""
import math

import pytest
import torch

from oracle import ref
from test_logprobs_gpu import U, f32, head, near, special

pytestmark = pytest.mark.gpu
SHARE = torch.tensor([0.4, 0.2, 0.1])


def bounds(z, ids, t, temperature=1.0, softcap=0.0, dl=1.0):
    """(row loss, its bound, gradient, its bound)"""
    tau, cap = f32(temperature), f32(softcap)
    x, td, V = z.double(), t.double(), z.shape[1]
    kw = dict(tail="bucket", temperature=tau, softcap=cap, reduction="none")
    per, grad = ref.distill_fwd(x, ids, td, **kw), ref.distill_bwd(x, ids, td, dloss=dl, **kw)
    s = ref.token_scores(x, tau, cap)
    m = s.max(1, keepdim=True).values
    D, p = s - m, torch.softmax(s - m, 1)
    q, _, r, ok = ref._teacher(ids.long(), td, V, "bucket", tau)
    hidden = torch.zeros(z.shape[0], V + 1, dtype=torch.bool).scatter(1, torch.where(ok, ids.long(), V), True)[:, :V]
    others = torch.where(hidden, -math.inf, s)
    lead = m - others.max(1, keepdim=True).values
    behind = torch.where(others == -math.inf, 0.0, -(others - others.max(1, keepdim=True).values))
    share = torch.softmax(others + (lead - m), 1)
    log_s = (torch.logsumexp(others + (lead - m), 1) - torch.logsumexp(D, 1))[:, None] - lead
    off, chain = cap * 2.0 ** -21 / tau, (V / 1024 + 24) * U
    mean = lambda w, x: torch.where(w > 0, w * x, 0.0).sum(1, keepdim=True)  # noqa: E731
    of_lse = chain + 5 * U * mean(p, D.abs()) + 3 * U * torch.logsumexp(D, 1)[:, None] + 2 * U + 2 * off
    up = lead.clamp(max=47)
    of_sum = chain + 5 * U * (mean(share, behind) + up) + 2 * off + 2 * U
    of_log_s = of_sum + 3 * U * (up + math.log(V)) + 5 * U * lead + off + 3 * U * log_s.abs() + of_lse
    q_log = torch.where(q > 0, td, 0.0)
    at = ids.long().clamp(0, V - 1)
    logp = torch.where(q > 0, (D - torch.logsumexp(D, 1, keepdim=True)).gather(1, at), 0.0)
    own = torch.where(q > 0, D.abs().gather(1, at), 0.0)
    of_q = q * (4 * U * q_log.abs() + 16 * U)
    of_r = of_q.sum(1, keepdim=True) + 10 * U
    r = r[:, None]
    r_log = torch.where(r > 0, r.log(), 0.0).abs()
    bound = (of_q * (q_log - logp).abs() + q * (of_lse + off + 5 * U * own + 12 * U * (q_log.abs() + logp.abs()))).sum(1, keepdim=True)
    bound = bound + torch.where(r > 0, of_r * (r_log + log_s.abs() + 1) + r * (of_log_s + 6 * U * (r_log + log_s.abs())), 0.0)
    raw = torch.where(p > 0, p * (of_lse + off + 5 * U * D.abs() + 12 * U + of_r), 0.0)
    raw = raw + torch.where(share > 0, share * (of_r + r * (of_sum + 2 * off + 5 * U * (behind + up) + 12 * U)), 0.0)
    raw = raw.scatter_add(1, at, of_q + 4 * U * q)
    if softcap:
        raw = raw + 2.0 ** -20 * (p + r * share).scatter_add(1, at, q)
    # An exponential below 2^-126 may be flushed; it is multiplied by (sum q + r) / S and by r / S', S' being at least exp(-up), its largest term, where it is taken against a score `up`
    # above m'.  (At a lead of 20 scores r / S' is 1.5e8: 1e-38 flushed is 1.5e-30 of a probability, 10^-28 of the gradient's largest number.)
    flushed = 2.0 ** -126 * (1 + r * up.exp())
    gbound = (raw + flushed) * abs(dl) / tau + torch.finfo(z.dtype).eps / 2 * (1 + 2.0 ** -10) * grad.abs() + 2.0 ** -120
    return per, bound[:, 0] + 8 * U * per.abs() + 4 * U, grad, gbound


LEADS = [0.0, 30.0, 46.0, 47.0, 60.0, 75.0, 85.0, 120.0, 8192.0]


def make(V, dtype, leads, std=2.5, seed=0):
    """A row to a lead, one of half its tokens masked, and one that is left out; the teacher's tokens are the row's first, its last and one between."""
    g = torch.Generator().manual_seed(seed + V)
    n = len(leads) + 2
    z = torch.randn(n, V, generator=g) * std
    z[n - 2, V // 4: 3 * V // 4] = -math.inf
    ids = torch.tensor([0, V - 1, V // 3]).repeat(n, 1)
    top = z.max(1, keepdim=True).values
    z.scatter_(1, ids, top + torch.tensor([*leads, 85.0, 85.0])[:, None] + torch.tensor([[0.0, -0.5, -1.0]]))
    ids[n - 1, 0] = -1
    t = SHARE.log().repeat(n, 1)
    t[1] = torch.tensor([0.6, 0.3, 0.1]).log()  # (nothing is left for the others)
    return z.to(dtype), ids.to(torch.int32), t


# rows held by 256, 512 and 1024 threads, in shares, and streamed by whole workgroups
FORMS = [(11, 1000), (11, 50304), (200, 150001), (3, 262147), (300, 262147), (405, 20001)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,V", FORMS)
def test_the_others_far_behind(dtype, T, V):
    from olmax_amd import ops
    print(f"[case] tail {T} {V}", flush=True)
    z, ids, t = make(V, dtype, LEADS)
    n = z.shape[0]
    if T < n:  # few rows: those of the largest leads
        z, ids, t = z[-T - 2:-2], ids[-T - 2:-2], t[-T - 2:-2]
        n = T
    per, bound, grad, gbound = bounds(z, ids, t)
    copies = (T + n - 1) // n
    many = lambda a: a.cuda().repeat(copies, 1)[:T]  # noqa: E731
    rows, ids, t = many(z), many(ids), many(t)
    loss, d = ops.distill(rows, ids, t, tail="bucket", reduction="none")
    alone, _ = ops.distill(rows, ids, t, tail="bucket", reduction="none", want_grad=False)
    for i in range(0, T, 1 if T < 50 else 7):
        near(loss[i], per[i % n], bound[i % n], f"row loss {i}")
        near(alone[i], per[i % n], bound[i % n], f"row loss alone {i}")
        near(d[i], grad[i % n], gbound[i % n], f"dlogits {i}")
    mean, dm = ops.distill(rows, ids, t, tail="bucket", inplace=True)
    kept = (ids[:, 0] >= 0).sum().item()
    want = per[torch.arange(T) % n]
    near(mean, want.sum() / kept, bound[torch.arange(T) % n].sum() / kept + (T / 1024 + 12) * U * want.abs().sum() / kept, "mean")
    for i in (0, T // 2, T - 1):
        near(dm[i], grad[i % n] / kept, gbound[i % n] / kept + 3 * U * grad[i % n].abs() / kept + 2.0 ** -120, f"dlogits of the mean {i}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,V", FORMS)
@pytest.mark.parametrize("temperature,softcap", [(0.05, 0.0), (0.25, 30.0), (4.0, 0.0)])
def test_small_leads_at_a_temperature(dtype, T, V, temperature, softcap):
    """A lead of 7 logits is 140 scores at a temperature of 0.05."""
    from olmax_amd import ops
    z, ids, t = make(V, dtype, [1.0, 3.0, 4.0, 7.0, 20.0], std=1.0)
    z, ids, t = z[:5], ids[:5], t[:5]
    kw = dict(temperature=temperature, softcap=softcap)
    per, bound, grad, gbound = bounds(z, ids, t, dl=-3.0, **kw)
    many = lambda a: a.cuda().repeat((T + 4) // 5, 1)[:T]  # noqa: E731
    loss, d = ops.distill(many(z), many(ids), many(t), tail="bucket", reduction="none", dloss=-3.0, **kw)
    alone, _ = ops.distill(many(z), many(ids), many(t), tail="bucket", reduction="none", want_grad=False, **kw)
    for i in range(0, T, 1 if T < 50 else 7):
        near(loss[i], per[i % 5], bound[i % 5], f"row loss {i}")
        near(alone[i], per[i % 5], bound[i % 5], f"row loss alone {i}")
        near(d[i], grad[i % 5], gbound[i % 5], f"dlogits {i}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 3.0])
@pytest.mark.parametrize("V,copies", [(997, 1), (60001, 1), (60001, 80), (262147, 1)])
def test_masked_rows(dtype, temperature, V, copies):
    """Others at the type's lowest value, at minus infinity, 8192 behind, about -1e30: all rows that have others at all."""
    from olmax_amd import ops
    z, first = special(V, dtype)
    z[12], z[13] = 1e30, -3e38
    z[13, 5] = torch.finfo(dtype).max / 2
    first[12], first[13] = 7, 5
    ids = torch.stack([first, (first + 3) % V], 1)
    t = torch.tensor([[-0.25, -math.inf]]).repeat(14, 1)
    kw = dict(tail="bucket", temperature=temperature, reduction="none")
    loss, d = ops.distill(z.cuda().repeat(copies, 1), ids.cuda().repeat(copies, 1), t.cuda().repeat(copies, 1), **kw)
    rows = [1, *range(3, 14)]
    per, bound, grad, gbound = bounds(z[rows], ids[rows], t[rows], temperature)
    for c in range(min(copies, 4)):
        one, dz = loss[14 * c:14 * c + 14].cpu(), d[14 * c:14 * c + 14].cpu()
        near(one[rows], per, bound, "row losses")
        near(dz[rows], grad, gbound, "dlogits")
        assert one[0] == 0 and (dz[0] == 0).all()
        # one token and no other: infinitely far off, and nothing to pull on
        assert one[2] == math.inf and torch.isfinite(dz[2]).all() and (dz[2][torch.arange(V) != V // 2] == 0).all()


@pytest.mark.parametrize("T,d,V", [(5, 256, 4096), (63, 1024, 8001), (130, 256, 40007), (300, 320, 1030), (513, 1024, 5000)])
@pytest.mark.parametrize("lead,temperature", [(60.0, 1.0), (90.0, 1.0), (7.0, 0.05)])
def test_lmhead(T, d, V, lead, temperature):
    """Each token's state is some of the head's own row of its teacher's token, which leads by about `lead`.  dW of the others comes from the tail alone: its norm, as those of all of
    dh and dW, is off by two roundings to bf16, 2^-8, and by what the logits' fp32 sums differ by in the exponents, 4 sqrt(d) u sum |h w| / temperature, small against that."""
    from olmax_amd import ops
    h, W, _ = head(T, d, V)
    at = torch.arange(T, device="cuda") % 40
    h = (W[at].float() * (lead / (W[at].float() ** 2).sum(1, keepdim=True)) + h.float() * 0.1).bfloat16()
    z = (h.double() @ W.double().t()).cpu()
    ids, t = at[:, None].to(torch.int32).cpu(), torch.full((T, 1), math.log(0.5))
    kw = dict(tail="bucket", temperature=f32(temperature))
    want, dz = ref.distill_fwd(z, ids, t.double(), **kw), ref.distill_bwd(z, ids, t.double(), **kw).cuda()
    loss, dh, dW = ops.lmhead_distill(h, W, ids.cuda(), t.cuda(), tail="bucket", temperature=temperature)
    of_z = 4 * math.sqrt(d) * U * (h.double().abs() @ W.double().abs().t()).max().item() / f32(temperature)
    assert of_z < 2.0 ** -9
    assert abs(loss.item() - want.item()) <= 3 * of_z + 2.0 ** -19 * (1 + abs(want.item()))
    wh, wW = dz @ W.double(), dz.t() @ h.double()
    for got, w in ((dh, wh), (dW, wW), (dW[40:], wW[40:])):
        assert (got.double() - w).norm() <= (2.0 ** -8 + 4 * of_z) * w.norm()
