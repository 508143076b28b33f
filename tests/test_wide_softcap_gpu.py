"""Soft-caps far above the logits: scores are nearly the logits, and as exact as those.

Up to a soft-cap of 64 a score is off by softcap 2^-21 / temperature.  Above, of a score with |x| < softcap / 4 the scaled logit (the factor and the product), the sum with its series'
share and that share itself (0.021 of it at most, to a few roundings, its end left off 0.14 u) lose 4 u of it, u = 2^-24; further out tanh is off by 2^-22, of at least 0.2449, and its factor
by three roundings: under 2^-19.  Two scores make a difference; the rest is as without a soft-cap, on scores that 64 bits hold exactly."""
import math

import pytest
import torch

from oracle import ref
from test_distill_tail_gpu import bounds
from test_logprobs_gpu import U, Row, f32, head, make, near, score_grads, teacher

pytestmark = pytest.mark.gpu
CAPS = [64.0, 65.0, 200.0, 1000.0, 1e4, 1e6, 1e30]
FORMS = [(7, 1000), (7, 4099), (3, 60001), (300, 1003), (300, 20001)]


def off(z, temperature, softcap):
    """[T]: what a score of each row is off by at most"""
    if softcap <= 64:
        return torch.full((z.shape[0],), softcap * 2.0 ** -21 / temperature, dtype=torch.float64)
    s = ref.token_scores(z.double(), temperature, softcap).abs()
    return torch.where(z.double().abs() < softcap / 4, 4 * U * s, 2.0 ** -19 * s).max(1).values


def slope(z, temperature, softcap):
    return (1 - torch.tanh(z.double() / softcap) ** 2) / temperature


def check(r, s, of_s, targets, rows):
    lp, ent, best, ids = ref.token_logprobs_fwd(s, targets, top=0 if r.top_ids is None else r.top_ids.shape[1])
    b = Row(s)
    near(r.logprobs[rows], lp, b.of_lp(lp) + 2 * of_s, "logprobs")
    near(r.entropy[rows], ent, b.of_entropy + 2 * of_s * (1 + b.first + b.lse), "entropy")
    if r.top_ids is not None:
        near(r.top_logprobs[rows], best, b.of_lp(best) + 2 * of_s[:, None], "top_logprobs")
    return b, ids


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,V", FORMS)
@pytest.mark.parametrize("softcap", CAPS)
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_scores_and_their_gradients(dtype, T, V, softcap, temperature):
    from olmax_amd import ops
    print(f"[case] wide soft-cap {softcap} {T} {V}", flush=True)
    n = min(T, 7)
    z, targets = make(n, V, dtype)
    z[0] *= 8.0  # past a quarter of the lowest caps
    tau, cap = f32(temperature), f32(softcap)
    s, of_s = ref.token_scores(z.double(), tau, cap), off(z, tau, cap)
    many = lambda a: a.repeat((T + n - 1) // n, *[1] * (a.dim() - 1))[:T].cuda()  # noqa: E731
    kw = dict(temperature=temperature, softcap=softcap)
    r = ops.token_logprobs(many(z), many(targets), top=5, **kw)
    last = torch.arange(T - n, T)
    for rows in (torch.arange(n), last):
        b, _ = check(r, s[rows % n], of_s[rows % n], targets[rows % n], rows)
    x = z.double()  # (the alternatives are those of the logits)
    assert torch.equal(r.top_ids[:n].cpu().long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :5])
    g, h = torch.linspace(-1, 2, n), torch.linspace(0.3, -0.2, n)
    got = ops.token_logprobs_bwd(many(z), many(targets), r.stats, many(g), dentropy=many(h), **kw)
    want = ref.token_logprobs_bwd(x, targets, g.double(), h.double(), temperature=tau, softcap=cap)
    b = Row(s)
    _, bound = score_grads(s, targets, g, h)
    gd, hd, logp = g.double().abs()[:, None], h.double().abs()[:, None], torch.where(b.p > 0, b.p.log(), 0.0).abs()
    column = lambda a: a[:, None]  # noqa: E731
    moved = b.p * (gd + hd * (logp + column(b.lse + b.first) + 1) + hd * column(1 + b.first + b.lse)) * column(2 * of_s)
    bound = (bound + moved) * slope(z, tau, cap) + (2.0 ** -20 + torch.finfo(dtype).eps / 2 * (1 + 2 ** -10)) * want.abs() + 2.0 ** -120
    near(got[:n], want, bound, "dlogits")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,V", [(7, 1000), (3, 262147), (5, 50304), (405, 20001)])
@pytest.mark.parametrize("softcap", [65.0, 1e4, 1e30])
def test_distillation(dtype, T, V, softcap):
    from olmax_amd import ops
    n = min(T, 7)
    z, _ = make(n, V, dtype)
    cap, of_s = f32(softcap), off(z, 1.0, f32(softcap))
    s = ref.token_scores(z.double(), 1.0, cap)
    ids, t = teacher(z, 9)
    many = lambda a: a.repeat((T + n - 1) // n, 1)[:T].cuda()  # noqa: E731
    kw = dict(tail="bucket", softcap=softcap, reduction="none")
    loss, d = ops.distill(many(z), many(ids), many(t), **kw)
    alone, _ = ops.distill(many(z), many(ids), many(t), want_grad=False, **kw)
    per, bound, grad, gbound = bounds(s, ids, t)
    near(loss[:n], per, bound + 4 * of_s, "row losses")
    near(alone[:n], per, bound + 4 * of_s, "row losses alone")
    q, _, rest, _ = ref._teacher(ids.long(), t.double(), V, "bucket", 1.0)
    p = torch.softmax(s, 1)
    others = p.scatter(1, ids.long(), 0.0)
    moved = (p + rest[:, None] * others / others.sum(1, keepdim=True)) * 2 * of_s[:, None]
    want = grad * slope(z, 1.0, cap)
    near(d[:n], want, (gbound + moved) * slope(z, 1.0, cap) + (2.0 ** -20 + torch.finfo(dtype).eps / 2 * (1 + 2 ** -10)) * want.abs() + 2.0 ** -120, "dlogits")


@pytest.mark.parametrize("T,d,V", [(5, 256, 4096), (256, 64, 70000), (300, 72, 50301), (40, 128, 50301)])
@pytest.mark.parametrize("softcap", [1000.0, 1e6])
def test_lmhead(T, d, V, softcap):
    from olmax_amd import ops
    h, W, t = head(T, d, V)
    r = ops.lmhead_logprobs(h, W, t, softcap=softcap)
    few = torch.arange(min(T, 40))
    z = (h[:40].double() @ W.double().t()).cpu()
    of_z = (4 * math.sqrt(d) * U * (h[:40].double().abs() @ W.double().abs().t()).max(1).values).cpu()
    check(r, ref.token_scores(z, 1.0, softcap), of_z + off(z, 1.0, softcap), t[:40].cpu(), few)
    g = torch.randn(T, device="cuda")
    dh, dW = ops.lmhead_logprobs_bwd(h, W, t, r.stats, g, dentropy=g * 0.1, softcap=softcap)
    z = h.double() @ W.double().t()
    dz = ref.token_logprobs_bwd(z.cpu(), t.cpu(), g.cpu().double(), g.cpu().double() * 0.1, softcap=softcap).cuda()
    for got, want in ((dh, dz @ W.double()), (dW, dz.t() @ h.double())):
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()
