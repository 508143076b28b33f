"""Log probabilities, policy-gradient and distillation steps through the whole model, against the cross entropy's path and against the same calls' definitions."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(layer_type="default", tied=False, softcap=0.0, vocab=1000, batch=2, seq=96, ac=None, seed=0):
    from olmax_amd import TransformerConfig
    cfg = TransformerConfig(vocab_size=vocab, d_model=256, hidden_size=512, num_layers=2, n_heads=2, head_dim=128, layer_type=layer_type, tie_embeddings=tied,
                            final_logit_softcap=softcap, layer_ac_policy=ac)
    m = cfg.build(batch_size=batch, sequence_length=seq, seed=seed)
    m.master.mul_(2.0)  # a distribution that is not flat
    m.sync_working_copy()
    g = torch.Generator().manual_seed(seed + 1)
    ids = torch.randint(0, vocab, (batch * seq,), generator=g, dtype=torch.int32).cuda()
    labels = torch.randint(0, vocab, (batch * seq,), generator=g, dtype=torch.int32).cuda()
    labels[5:9] = -100
    return m, ids, labels


KINDS = [dict(), dict(tied=True, softcap=5.0), dict(layer_type="gemma", ac="nothing_saveable", vocab=70000, seq=128), dict(vocab=1003, batch=1, seq=300, ac="nothing_saveable")]


def same(a, b, bound):
    """Gradient buffers that come from logits of another precision."""
    for n in a:
        x, y = a[n].double(), b[n].double()
        assert (x - y).norm() <= bound * y.norm() + 1e-30, (n, ((x - y).norm() / y.norm()).item())


@pytest.mark.parametrize("kind", KINDS, ids=lambda k: "-".join(map(str, k.values())) or "plain")
def test_the_cross_entropys_step(kind):
    """-mean(logprobs) is the cross entropy, whose logits are rounded to bf16 (2^-9 of themselves, under 16 here: 2^-5 of a row's loss at most, averaged over 180 rows of
    either sign 2^-8); gradients by logprobs_grads and by distilling from the label alone are the cross entropy's, to the 2^-6 that probabilities of such logits differ by,
    and each other's to the two roundings of bf16 that they do not share, 2^-7 behind two layers."""
    m, ids, labels = build(**kind)
    counted = int((labels != -100).sum())
    loss = m.loss_and_grads(ids, labels).item()
    want = m.named_gradients()
    want = {n: g.clone() for n, g in want.items()}
    r = m.token_logprobs(ids, labels, top=4)
    assert abs(-r.logprobs.sum().item() / counted - loss) < 2 ** -8 * (1 + loss)
    m.logprobs_grads(ids, labels, r.stats, torch.full_like(r.logprobs, -1.0 / counted))
    policy = {n: g.clone() for n, g in m.named_gradients().items()}
    same(policy, want, 2 ** -6)
    mine = m.distill_loss_and_grads(ids, torch.where(labels < 0, -1, labels)[:, None].contiguous(), torch.zeros(labels.numel(), 1, device="cuda")).item()
    assert abs(mine + r.logprobs.sum().item() / counted) < 2 ** -19 * (1 + loss)
    same(m.named_gradients(), policy, 2 ** -7)
    # greedy tokens are the rows' best
    best = m.token_logprobs(ids, r.top_ids[:, 0].contiguous().where(labels >= 0, labels))
    assert (best.logprobs - r.top_logprobs[:, 0].where(labels >= 0, torch.zeros_like(best.logprobs))).abs().max() < 2 ** -18 * 16
    assert (r.top_ids[5:9] == -1).all() and (r.top_logprobs[:, :-1] >= r.top_logprobs[:, 1:]).all()


def test_a_teacher_a_student_and_a_policy_step():
    """A teacher's pass, steps of distillation with the optimizer, a policy step with an entropy bonus: everything runs and stays finite.  The policy's gradients are linear in
    the cotangents: with both doubled (a power of two: exact but for what atomics add up in another order) twice as large, and the sum of what each gives alone to three roundings
    of bf16 behind two layers, 2^-6."""
    teacher, ids, labels = build(seed=3)
    student, _, _ = build(seed=4)
    notes = teacher.token_logprobs(ids, top=32)
    old = student.master.clone()
    for step in range(1, 4):
        loss = student.distill_loss_and_grads(ids, notes.top_ids, notes.top_logprobs, tail="bucket")
        assert torch.isfinite(loss) and all(torch.isfinite(g).all() for g in student.named_gradients().values())
        student.adamw_step(step=step, lr=1e-3)
    assert torch.isfinite(student.master).all() and not torch.equal(old, student.master)
    r = student.token_logprobs(ids, labels)
    g, h = torch.randn_like(r.logprobs), torch.randn_like(r.entropy) * 0.1
    grads = {}
    for name, a, b in (("both", g, h), ("twice", 2 * g, 2 * h), ("targets", g, torch.zeros_like(h)), ("entropy", torch.zeros_like(g), h), ("alone", g, None)):
        student.logprobs_grads(ids, labels, r.stats, a, dentropy=b)
        grads[name] = {n: x.clone() for n, x in student.named_gradients().items()}
    same({n: x / 2 for n, x in grads["twice"].items()}, grads["both"], 2 ** -16)
    same({n: x + grads["entropy"][n] for n, x in grads["targets"].items()}, grads["both"], 2 ** -6)
    same(grads["alone"], grads["targets"], 2 ** -16)


def test_refused_before_anything_is_launched():
    from olmax_amd import _lib
    m, ids, labels = build()
    m.grad_f32.fill_(7.0)
    for call in (lambda: m.token_logprobs(ids, labels, top=129), lambda: m.token_logprobs(ids, labels, temperature=0.0),
                 lambda: m.distill_loss_and_grads(ids, torch.zeros(192, 0, dtype=torch.int32, device="cuda"), torch.zeros(192, 0, device="cuda")),
                 lambda: m.distill_loss_and_grads(ids, labels[:, None], torch.zeros(192, 1, device="cuda"), tail="none"),
                 lambda: m.logprobs_grads(ids, labels, torch.zeros(192, 2, device="cuda"), torch.zeros(192, device="cuda"))):
        with pytest.raises(_lib.OlmaxHipError):
            call()
    torch.cuda.synchronize()
    assert (m.grad_f32 == 7).all()
    with pytest.raises(ValueError):
        m.token_logprobs(ids, labels[:-1])
