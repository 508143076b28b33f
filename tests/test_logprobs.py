"""The plain forms of log probabilities and distillation against autograd, differences and torch's own routines, and what the entry points refuse.  No GPU needed."""
import ctypes
import math

import pytest
import torch

from oracle import ref


def _rows(T, V, seed=0):
    return torch.randn(T, V, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 3


@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (0.7, 0.0), (2.0, 5.0)])
def test_score_gradient_is_autograds(temperature, softcap):
    """float64 through some 20 operations: 1e-12 of the largest."""
    z = _rows(5, 40).requires_grad_()
    t = torch.tensor([3, 39, -100, 40, 0])  # ignored, out of range
    g, h = torch.randn(5, dtype=torch.float64), torch.randn(5, dtype=torch.float64)
    lp, ent, _, _ = ref.token_logprobs_fwd(z, t, temperature=temperature, softcap=softcap)
    ((lp * g).sum() + (ent * h).sum()).backward()
    want = ref.token_logprobs_bwd(z.detach(), t, g, h, temperature=temperature, softcap=softcap)
    assert (z.grad - want).abs().max() < 1e-12
    assert (want[2] == 0).all()


def test_scores_are_torchs():
    z = _rows(6, 100)
    t = torch.arange(6)
    lp, ent, best, ids = ref.token_logprobs_fwd(z, t, top=7)
    d = torch.distributions.Categorical(logits=z)
    assert (lp - d.log_prob(t)).abs().max() < 1e-12 and (ent - d.entropy()).abs().max() < 1e-12
    v, i = torch.topk(torch.log_softmax(z, 1), 7, dim=1)
    assert torch.equal(i, ids) and (v - best).abs().max() < 1e-12


def test_ties_and_rows_of_nothing():
    z = torch.zeros(3, 6, dtype=torch.float64)
    z[1] = -math.inf
    z[2, :5] = torch.tensor([-math.inf, 1.0, -math.inf, 1.0, 2.0])
    z[2, 5] = -math.inf
    lp, ent, best, ids = ref.token_logprobs_fwd(z, torch.tensor([0, 0, 4]), top=5)
    assert ids.tolist() == [[0, 1, 2, 3, 4], [0, 1, 2, 3, 4], [4, 1, 3, 0, 2]]
    assert abs(ent[0] - math.log(6)) < 1e-12 and ent[1] == 0 and lp[1] == -math.inf and best[2, 3] == -math.inf


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (2.0, 6.0)])
def test_distill_gradient_is_autograds_and_the_differences(tail, reduction, temperature, softcap):
    z = _rows(4, 30).requires_grad_()
    t, ids = torch.topk(torch.log_softmax(_rows(4, 30, 1), 1), 6, dim=1)
    ids[1, 3] = ids[1, 0]  # named again
    ids[2, 2] = -1
    ids[3, 0] = -1         # left out
    kw = dict(tail=tail, temperature=temperature, softcap=softcap, reduction=reduction)
    dl = torch.tensor([1.0, -2.0, 0.5, 3.0], dtype=torch.float64) if reduction == "none" else torch.tensor(1.5, dtype=torch.float64)
    (ref.distill_fwd(z, ids, t, **kw) * dl).sum().backward()
    want = ref.distill_bwd(z.detach(), ids, t, dloss=dl, **kw)
    assert (z.grad - want).abs().max() < 1e-12 and (want[3] == 0).all()
    assert want[:3].sum(1).abs().max() < 1e-12 or softcap  # a constant added to a row changes nothing
    f = lambda x: (ref.distill_fwd(x, ids, t, **kw) * dl).sum().item()  # noqa: E731
    for r, c in ((0, int(ids[0, 0])), (1, 5), (2, 17)):  # central differences: h^2 of the third derivative, 2^-52 / h
        e = torch.zeros_like(want)
        e[r, c] = 1e-5
        assert abs((f(z.detach() + e) - f(z.detach() - e)) / 2e-5 - want[r, c]) < 1e-8


def test_distill_is_kl_div():
    """All tokens named: both tails are the divergence of two softmaxes; the bucket of one token is that of two events."""
    z, u = _rows(3, 8), _rows(3, 8, 1)
    t, ids = torch.topk(torch.log_softmax(u, 1), 8, dim=1)
    want = torch.nn.functional.kl_div(torch.log_softmax(z, 1), torch.log_softmax(u, 1), reduction="none", log_target=True).sum(1)
    assert (ref.distill_fwd(z, ids, t, reduction="none") - want).abs().max() < 1e-12
    p, q = torch.softmax(z, 1), torch.softmax(u, 1)
    a, b = p.gather(1, ids[:, :1])[:, 0], q.gather(1, ids[:, :1])[:, 0]
    two = b * (b / a).log() + (1 - b) * ((1 - b) / (1 - a)).log()
    assert (ref.distill_fwd(z, ids[:, :1], t[:, :1], tail="bucket", reduction="none") - two).abs().max() < 1e-12


def _lib():
    from olmax_amd import _lib
    if not _lib.lib_path().exists():
        pytest.skip("libolmax_hip.so not built")
    return _lib


# a valid call's arguments by name, on addresses that are never read: each refusal changes one of them, and is found before any launch
P = 1 << 20
CALLS = {
    "olmax_token_logprobs": dict(stream=None, logits=P, targets=P, logprobs=P, entropy=P, stats=P, top_ids=P, top_logprobs=P, workspace=P, workspace_bytes=1 << 40, T=4, V=100,
                                 ld=100, top=5, logits_f32=0, ignore_index=-100, temperature=1.0, softcap=0.0),
    "olmax_token_logprobs_bwd": dict(stream=None, logits=P, targets=P, stats=P, dlogprobs=P, dentropy=None, dlogits=2 * P, T=4, V=100, ld=100, ldd=100, logits_f32=0,
                                     ignore_index=-100, temperature=1.0, softcap=0.0),
    "olmax_distill": dict(stream=None, logits=P, dlogits=2 * P, top_ids=P, top_logprobs=P, loss=P, dloss_rows=None, workspace=P, workspace_bytes=1 << 40, T=4, V=100, k=5, ld=100,
                          ldd=100, logits_f32=0, tail=0, temperature=1.0, softcap=0.0, dloss=1.0, reduction=0),
    "olmax_lmhead_logprobs": dict(stream=None, h=P, W=P, targets=P, logprobs=P, entropy=P, stats=P, top_ids=P, top_logprobs=P, workspace=P, workspace_bytes=1 << 40, T=4, d=64,
                                  V=100, top=5, ignore_index=-100, temperature=1.0, softcap=0.0),
    "olmax_lmhead_logprobs_bwd": dict(stream=None, h=P, W=P, targets=P, stats=P, dlogprobs=P, dentropy=None, dh=P, dW=P, workspace=P, workspace_bytes=1 << 40, T=4, d=64, V=100,
                                      ignore_index=-100, temperature=1.0, softcap=0.0, dw_f32=0),
    "olmax_lmhead_distill": dict(stream=None, h=P, W=P, top_ids=P, top_logprobs=P, loss=P, dh=P, dW=P, workspace=P, workspace_bytes=1 << 40, T=4, d=64, V=100, k=5, tail=0,
                                 temperature=1.0, softcap=0.0, dloss=1.0, dw_f32=0),
}
ARG, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -5
REFUSED = [(name, change, code) for name, given in CALLS.items() for change, code in (
    *(({n: None}, ARG) for n in ("logits", "h", "W", "targets", "entropy", "stats", "dlogprobs", "dlogits_out", "top_ids", "top_logprobs", "loss") if n in given),
    ({"T": 0}, SHAPE), ({"V": 0}, SHAPE), ({"T": 1 << 24}, SHAPE), ({"V": 1 << 30, "ld": 1 << 30, "ldd": 1 << 30}, SHAPE), ({"V": 1 << 30, "d": 64}, SHAPE), ({"d": 0}, SHAPE), ({"ld": 99}, SHAPE), ({"ldd": 99}, SHAPE),
    ({"temperature": 0.0}, ARG), ({"temperature": -1.0}, ARG), ({"temperature": math.nan}, ARG), ({"temperature": math.inf}, ARG), ({"softcap": -1.0}, ARG),
    ({"softcap": math.nan}, ARG), ({"top": -1}, ARG), ({"top": 129}, ARG), ({"top": 101}, ARG), ({"k": 0}, ARG), ({"k": 129}, ARG), ({"tail": 2}, ARG),
    ({"tail": 1, "V": 1 << 20, "ld": 1 << 20, "ldd": 1 << 20}, ARG), ({"reduction": 3}, ARG), ({"dloss_rows": P}, ARG), ({"logits": P + 1}, ALIGN),
    ({"logits": P, "dlogits": P, "ldd": 104}, ARG), ({"logits": P, "dlogits": P + 2}, ARG), ({"logits": P, "dlogits": P + 206}, ARG),
    ({"logits": P, "dlogits": P + 200, "ld": 199, "ldd": 199}, ARG), ({"logits": P + 400, "dlogits": P, "ld": 100, "ldd": 104}, ARG), ({"workspace_bytes": 8}, WORKSPACE), ({"workspace": P + 4}, WORKSPACE),
) if all(n in given for n in change)]


@pytest.mark.parametrize("name,change,code", REFUSED, ids=lambda v: str(v))
def test_refused_calls(name, change, code):
    lib = _lib()
    given = {**CALLS[name], **change}
    if name == "olmax_token_logprobs" and "workspace" in str(change):
        given.update(T=1, V=100000, ld=100000)  # a row in parts needs one
    rc = lib.typed(name)(*given.values())
    assert rc == code, lib.load().olmax_last_error_string()
    assert name.encode() in lib.load().olmax_last_error_string()


def test_workspace_queries():
    _lib()
    from olmax_amd import ops
    assert ops._size("olmax_token_logprobs_workspace_bytes", 4096, 50304, 20, 0) == 0
    assert 0 < ops._size("olmax_token_logprobs_workspace_bytes", 1, 128256, 128, 0) <= 64 * (128 * 8 + 12)
    assert ops._size("olmax_distill_workspace_bytes", 1000, 5000, 8, 0) >= 4004
    for T, d, V in ((1, 64, 100), (2048, 4096, 100278)):
        n = ops._size("olmax_lmhead_logprobs_bwd_workspace_bytes", T, d, V)
        assert n >= T * V * 2 and n % 256 == 0


def test_ops_refuse_cpu_tensors():
    from olmax_amd import _lib, ops
    z, t = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_lib.OlmaxHipError, match="CPU"):
        ops.token_logprobs(z, t)
    with pytest.raises(_lib.OlmaxHipError, match="CPU"):
        ops.distill(z, t[:, None], torch.zeros(2, 1))
    with pytest.raises(_lib.OlmaxHipError, match="CPU"):
        ops.lmhead_logprobs(z, z, t)


def test_argument_checks():
    """The helpers behind every wrapper, on CPU tensors."""
    from olmax_amd import _lib, ops
    z = torch.zeros(4, 16, dtype=torch.bfloat16)
    bad = _lib.OlmaxHipError
    assert ops._logits(z[:, :9])[1] == 16 and ops._logits(z[:1, :9].expand(1, 9))[1] >= 9
    for t in (z[0], z.t(), z.half(), z[:1, :].expand(4, 16), z.int()):
        with pytest.raises(bad):
            ops._logits(t)
    with pytest.raises(bad):
        ops._logits(z, z[:, :9])
    with pytest.raises(bad):
        ops._logits(z.float(), z)
    for t in (torch.zeros(4, 1), torch.zeros(3), torch.zeros(8)[::2], torch.zeros(4, dtype=torch.float64)):
        with pytest.raises(bad):
            ops._row_of(t, 4, "dlogprobs")
    with pytest.raises(bad):
        ops._outputs(4, torch.zeros(4, dtype=torch.int64), 0, z)
    for top in (-1, 129, 1 << 40):
        with pytest.raises(bad):
            ops._outputs(4, None, top, z)
    ids, t = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    assert ops._teacher(ids, t, 4) == 3
    for a, b in ((ids.long(), t), (ids[:3], t[:3]), (ids, t[:, :2]), (ids, t.double()), (ids[:, ::2], t[:, ::2])):
        with pytest.raises(bad):
            ops._teacher(a, b, 4)
    with pytest.raises(bad):
        ops._tail("drop")
    w = torch.zeros(9, 16, dtype=torch.bfloat16)
    assert ops._head(z, w) == (4, 16, 9)
    for a, b in ((z.float(), w), (z, w.float()), (z[:, ::2], w[:, :8].contiguous()), (z, w[:, :8].contiguous()), (z[0], w)):
        with pytest.raises(bad):
            ops._head(a, b)


def test_rows_that_are_held_stay_in_registers(tmp_path):
    """Nor do the products with a row's softmax in their epilogue spill, or the scores."""
    import test_spills
    got = {n: v for n, v in test_spills.kernels(tmp_path).items() if any(k in n for k in ("distill_", "score_", "gemm_head_kernel"))}
    assert len(got) >= 40
    assert not any(got.values()), {n: v for n, v in got.items() if v}
