"""Products whose operands' rows are 2^25 elements and more apart, where the offset of a row within a tile has no room in 32 bits of bytes."""
import math

import pytest
import torch

from oracle import ref

pytestmark = pytest.mark.gpu
LONG = 2 ** 25 + 64


@pytest.mark.parametrize("al,bl", [(0, 0), (0, 1), (1, 1), (1, 0)])
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("tile", [0, 128, 256])
def test_products_of_views(al, bl, both, tile):
    """Whatever tile is asked for, the kernel that counts in 64 bits runs.  Two roundings to bf16 at most (2^-9 each, relative to the whole), as fp32 sums lose far less."""
    from olmax_amd import _lib, ops
    from test_gemm_choice_gpu import recorded
    M, N, K = 256, 512, 128
    print(f"[case] long rows a{al} b{bl} both {both} tile {tile}", flush=True)
    buffer = torch.empty(512, LONG, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    shape = lambda rows, layout: (K, rows) if layout else (rows, K)  # noqa: E731
    a, b = (torch.randn(*shape(n, l), device="cuda", generator=g).bfloat16() for n, l in ((M, al), (N, bl)))
    views = [buffer[:t.shape[0], at:at + t.shape[1]] for t, at in ((a, 64), (b, LONG - 512))]
    for v, t in zip(views, (a, b)):
        v.copy_(t)
    got = []
    _lib.load().olmax_gemm_set_tile(tile)
    try:
        keys = recorded(lambda: got.append(ops.gemm(views[0], views[1] if both else b, a_layout=al, b_layout=bl)))
    finally:
        _lib.load().olmax_gemm_set_tile(0)
    assert [key & 0xfff for key, *_ in keys] == [64], keys
    want = (a.double().t() if al else a.double()) @ (b.double() if bl else b.double().t())
    assert (got[0].double() - want).norm() <= 2.0 ** -8 * want.norm()


def test_lmhead_of_a_vocabulary_beyond_them():
    """Scores and gradients of three tokens over 2^25 + 64 logits, whose products are padded to tiles; dh and dW to two roundings to bf16, as elsewhere."""
    from olmax_amd import ops
    T, d, V = 3, 256, LONG
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn(T, d, device="cuda", generator=g).bfloat16()
    W = (torch.randn(V, d, device="cuda", generator=g) * 2 / math.sqrt(d)).bfloat16()
    t = torch.tensor([V - 1, 5, 2 ** 24 + 3], dtype=torch.int32, device="cuda")
    r = ops.lmhead_logprobs(h, W, t)
    c = torch.tensor([1.0, -2.0, 0.5], device="cuda")
    dh, dW = ops.lmhead_logprobs_bwd(h, W, t, r.stats, c)
    step = 2 ** 21
    z = torch.cat([h.double() @ W[i:i + step].double().t() for i in range(0, V, step)], 1)
    logp = ref._log_softmax(z)
    # sums of 2^25 exponentials: 2^25 / 1024 additions of a thread, 2^-24 each, at most (see the bounds of token_logprobs), and the logits' own 2^-17
    assert (r.logprobs.double() - logp.gather(1, t.long()[:, None])[:, 0]).abs().max() < 2.0 ** -9 + 2.0 ** -16
    dz = -c.double()[:, None] * logp.exp()
    dz[torch.arange(T), t.long()] += c.double()
    wh = sum(dz[:, i:i + step] @ W[i:i + step].double() for i in range(0, V, step))
    assert (dh.double() - wh).norm() <= 2.0 ** -8 * wh.norm()
    off = sum((dW[i:i + step].double() - dz[:, i:i + step].t() @ h.double()).norm() ** 2 for i in range(0, V, step))
    size = sum((dz[:, i:i + step].t() @ h.double()).norm() ** 2 for i in range(0, V, step))
    assert off.sqrt() <= 2.0 ** -8 * size.sqrt()
    ones = dW[t.long()].double() - dz[:, t.long()].t() @ h.double()
    assert ones.norm() <= 2.0 ** -8 * (dz[:, t.long()].t() @ h.double()).norm()
