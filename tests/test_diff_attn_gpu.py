"""GPU parity tests of differential attention and its gradients against the plain forms in 64 bits.

Tolerances count roundings; h = 2^-8 is bf16's half step, u = 2^-24.
Scores: the D products of a pair are added in fp32, at most D + 4 roundings of u A, A the largest sum of |q||k| / sqrt(D) that the row sees; the exponent is rounded
once (at most 2 u of |s| and |lse|, both within A + ln S), an exponential and its scale are off by 4 u.  So a probability is off by e = u (D + 16 + (D + 12) A + 4 ln S) of itself at most, and so is a log-normaliser, absolutely, with
2 u of itself and 16 u of a sum of positive numbers in pairs and (a tile of 64 keys at a time) S / 64 u.
o: a probability is rounded to bf16 in front of its product, h, and the result is, h; products are added in fp32, S u of the sum of the absolute ones: (h + 2 e + S u) (P_1 + |lam| P_2) |v| + h |o|.
Gradients take o, o2 (rounded to bf16 here) and lse (to fp32): delta_1 is off by d_1 = (h + 2D u) |do| (|o| + 2 |lam| |o2|), delta_2 by d_2 = (h + 2D u) |do| |o2|, dP by 2D u |do||v| and
(up to 512 tokens it is the kernel's own sum of P dP, off by e + (2D + S) u of P |do||v|), and
dS = P (dP - delta) by that and by e of itself, lse's rounding u |lse| in e; then h of itself in front of its products.  dlam is summed in fp32 from P_2 and dP: e + 2D u + (S + 1024) u of P_2 |do||v|."""
import math

import pytest
import torch

from oracle import ref

pytestmark = pytest.mark.gpu
H8, U = 2.0 ** -8 * (1 + 2 ** -7), 2.0 ** -24
BF = torch.bfloat16


def ops():
    from olmax_amd import ops
    return ops


def make(B, S, H, KH, D, seed=0, shared=False, scale=1.3):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, s=1.0: (torch.randn(B * S, n, generator=g) * s).to(BF)  # noqa: E731
    lam = torch.rand(1 if shared else H, generator=g) * 1.2 - 0.3
    return mk(H * 2 * D, scale), mk(KH * 2 * D, scale), mk(KH * 2 * D), lam, mk(H * 2 * D)


class Plain:
    """64-bit results and the bounds above."""

    def __init__(self, q, k, v, lam, do, window, own=False, **sizes):
        B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
        q, k, v, lam, do = (t.double() for t in (q, k, v, lam, do))
        self.o, self.o2, self.lse = ref.diff_attn_fwd(q, k, v, lam, window=window, **sizes)
        self.grads = ref.diff_attn_bwd(q, k, v, lam, do, window=window, **sizes)
        s, seen, qh, kh = ref._diff_maps(q, k, B, S, H, KH, D, window)
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        size = ref._diff_maps(q.abs(), k.abs(), B, S, H, KH, D, window)[0].masked_fill(~seen, 0.0)
        A = size.amax(-1)  # [B, H, 2, S]
        e = U * (D + 16 + (D + 12) * A + 4 * math.log(S + 1) + 2 * self.lse.abs())
        self.lse_room = e + U * (18 + S / 64 + 2 * self.lse.abs())
        group = lambda t: t.reshape(B, S, KH, 2 * D).permute(0, 2, 1, 3).repeat_interleave(H // KH, 1)  # noqa: E731
        heads = lambda t: t.reshape(B, S, H, 2 * D).permute(0, 2, 1, 3)  # noqa: E731
        rows = lambda t: t.permute(0, 2, 1, 3).reshape(B * S, -1)  # noqa: E731
        gather = lambda t: t.reshape(B, KH, H // KH, *t.shape[2:]).sum(2)  # noqa: E731
        w = lam.expand(H).abs()[:, None, None]
        e = e[..., None]
        rel = H8 + 2 * e + S * U
        far = (p[:, :, 0] * rel[:, :, 0] + w * p[:, :, 1] * rel[:, :, 1]) @ group(v).abs()
        self.o_room = rows(far) + H8 * self.o.abs() + 1e-30
        self.o2_room = rows((p[:, :, 1] * rel[:, :, 1]) @ group(v).abs()) + H8 * self.o2.abs() + 1e-30
        do_, v_ = heads(do), group(v)
        dp = (do_ @ v_.transpose(-1, -2))[:, :, None]
        big = (do_.abs() @ v_.abs().transpose(-1, -2))[:, :, None]
        delta = (p * dp).sum(-1, keepdim=True)
        o_, o2_ = heads(self.o).abs(), heads(self.o2).abs()
        d2 = (H8 + 2 * D * U) * (do_.abs() * o2_).sum(-1)
        d1 = (H8 + 2 * D * U) * (do_.abs() * (o_ + 2 * w * o2_)).sum(-1)
        if own:  # from the kernel's own outputs
            r, r2 = heads(self.o_room), heads(self.o2_room)
            d2 = d2 + (do_.abs() * r2).sum(-1)
            d1 = d1 + (do_.abs() * (r + w * r2)).sum(-1)
            e = e + self.lse_room[..., None]
            rel = H8 + 2 * e + S * U
        off = torch.stack([d1, d2], 2)[..., None]
        if S <= 512:  # the kernel's own sums of P dP
            off = (p * big).sum(-1, keepdim=True) * (e + (2 * D + S) * U)
        ds = (p * (dp - delta)).abs()
        ds_room = (H8 + 2 * e) * ds + p * (off + 2 * D * U * big) * (1 + H8)
        both = torch.stack([torch.ones_like(w).expand(H, 1, 1), w], 1)  # [H, 2, 1, 1]
        ds, ds_room = ds * both * D ** -0.5, (ds_room + S * U * ds) * both * D ** -0.5
        self.dq_room = (ds_room @ kh.abs()).permute(0, 3, 1, 2, 4).reshape(B * S, -1)
        self.dk_room = gather(ds_room.transpose(-1, -2) @ qh.abs()).permute(0, 3, 1, 2, 4).reshape(B * S, -1)
        self.dv_room = rows(gather((p[:, :, 0] * rel[:, :, 0] + w * p[:, :, 1] * rel[:, :, 1]).transpose(-1, -2) @ do_.abs()))
        dl = (p[:, :, 1] * big[:, :, 0] * (e[:, :, 1] + (2 * D + S + 1024) * U)).sum((0, 2, 3))
        self.dlam_room = dl.sum().view(1) if lam.shape[0] != H else dl
        for name, want in zip(("dq_room", "dk_room", "dv_room"), self.grads):
            setattr(self, name, getattr(self, name) + H8 * want.abs() + 1e-30)


def near(got, want, room, what):
    got = got.cpu().double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - room
    assert (off <= 0).all(), (what, off.max().item(), off.argmax().item(), int((~(off <= 0)).sum()), got.flatten()[off.argmax()].item(), want.flatten()[off.argmax()].item())


def forward(x, sizes, window, **more):
    q, k, v, lam, do = (t.cuda() for t in x)
    return ops().diff_attn_fwd(q, k, v, lam, window=window, **sizes, **more)


def backward(x, plain, sizes, window, **more):
    q, k, v, lam, do = (t.cuda() for t in x)
    return ops().diff_attn_bwd(q, k, v, lam, plain.o.to(BF).cuda(), plain.o2.to(BF).cuda(), plain.lse.float().cuda(), do, window=window, **sizes, **more)


def check(r, p):
    near(r.lse, p.lse, p.lse_room, "lse")
    near(r.o, p.o, p.o_room, "o")
    if r.o2 is not None:
        near(r.o2, p.o2, p.o2_room, "o2")


def check_grads(g, p):
    for name, got, want in zip(("dq", "dk", "dv", "dlam"), g, p.grads):
        near(got, want, getattr(p, name + "_room"), name)


SHAPES = [  # B, S, H, KH, D, window, shared
    (1, 1, 1, 1, 32, None, False), (1, 1, 2, 1, 64, None, True), (2, 2, 2, 2, 64, None, False), (2, 33, 4, 2, 64, None, False), (1, 64, 2, 2, 32, None, False), (1, 65, 3, 3, 64, None, True),
    (3, 127, 4, 1, 32, None, False), (1, 128, 8, 8, 64, None, False), (1, 129, 3, 1, 64, None, False), (2, 300, 4, 2, 64, 100, False), (1, 257, 2, 1, 32, 0, False), (1, 200, 2, 2, 64, 1, True),
    (3, 130, 6, 2, 32, 64, False), (1, 700, 4, 4, 64, None, False), (1, 515, 16, 2, 32, 63, False), (1, 640, 8, 4, 64, 128, False), (5, 48, 10, 5, 64, 47, False), (1, 90, 4, 2, 64, 1000, False),
    (1, 1100, 2, 1, 64, None, True), (1, 1030, 8, 8, 64, 300, False),
    # grids that fill the GPU: forms of 128 queries and keys to a workgroup
    (41, 130, 16, 8, 64, None, False), (41, 130, 8, 8, 32, 100, True), (3, 300, 20, 20, 32, None, False), (3, 300, 40, 20, 64, None, False), (33, 65, 40, 20, 64, 0, False),
    # few rows, long chains: dealt to many workgroups and joined
    (1, 2111, 1, 1, 64, None, False), (2, 1600, 2, 1, 32, None, True), (1, 4103, 1, 1, 32, None, False), (1, 3001, 2, 2, 64, 2000, False), (1, 1000, 4, 1, 32, 500, False)]


@pytest.mark.parametrize("B,S,H,KH,D,window,shared", SHAPES)
def test_against_the_plain_form(B, S, H, KH, D, window, shared):
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D)
    x = make(B, S, H, KH, D, seed=S, shared=shared)
    p = Plain(*x, window, **sizes)
    r = forward(x, sizes, window)
    check(r, p)
    g = backward(x, p, sizes, window)
    check_grads(g, p)
    again = backward(x, p, sizes, window)
    assert all(torch.equal(a, b) for a, b in zip(g, again))
    bare = forward(x, sizes, window, want_grad=False)
    assert bare.o2 is None and torch.equal(bare.o, r.o) and torch.equal(bare.lse, r.lse)


@pytest.mark.parametrize("scale", [0.0, 1e-3, 6.0])
def test_flat_and_sharp_maps(scale):
    sizes = dict(B=1, S=150, H=4, KH=2, D=64)
    x = make(**sizes, seed=5, scale=scale)
    p = Plain(*x, None, **sizes)
    check(forward(x, sizes, None), p)
    check_grads(backward(x, p, sizes, None), p)


@pytest.mark.parametrize("lam", [0.0, 1.0, -2.0, 30.0])
def test_weights(lam):
    sizes = dict(B=2, S=100, H=2, KH=1, D=32)
    q, k, v, _, do = make(**sizes, seed=6)
    x = (q, k, v, torch.tensor([lam]), do)
    p = Plain(*x, None, **sizes)
    check(forward(x, sizes, None), p)
    check_grads(backward(x, p, sizes, None), p)


@pytest.mark.parametrize("D", [32, 64])
def test_the_parts_of_fused_rows(D):
    """Queries, keys and values in the rows of one projection, gradients into the rows of another, outputs into wider rows; what is not theirs stays."""
    B, S, H, KH, W = 2, 150, 4, 2, 2 * D
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D)
    x = make(**sizes, seed=7)
    p = Plain(*x, 70, **sizes)
    wide = (H + 2 * KH) * W + 8
    qkv, dqkv, out = (torch.full((B * S, n), 5.0, dtype=BF, device="cuda") for n in (wide, wide, H * W + 64))
    parts = lambda t: (t[:, : H * W], t[:, H * W: (H + KH) * W], t[:, (H + KH) * W: (H + 2 * KH) * W])  # noqa: E731
    for a, b in zip(parts(qkv), x):
        a.copy_(b)
    lam, do = x[3].cuda(), x[4].cuda()
    r = ops().diff_attn_fwd(*parts(qkv), lam, window=70, **sizes, out=out[:, : H * W])
    check(r, p)
    dq, dk, dv = parts(dqkv)
    g = ops().diff_attn_bwd(*parts(qkv), lam, p.o.to(BF).cuda(), p.o2.to(BF).cuda(), p.lse.float().cuda(), do, window=70, **sizes, dq=dq, dk=dk, dv=dv)
    check_grads(g, p)
    assert out[:, H * W:].eq(5.0).all() and dqkv[:, -8:].eq(5.0).all() and qkv[:, -8:].eq(5.0).all()


@pytest.mark.parametrize("S,window", [(150, None), (1700, 1600)])
def test_rows_far_apart(S, window):
    """Operands and results as columns of rows whose distance is the largest that is taken, or that puts the last row behind 2^33 bytes: offsets that leave 32 bits, in bytes and in numbers."""
    sizes = dict(B=1, S=S, H=2, KH=1, D=32)
    ld, W = ((1 << 24) - 8 if S < 200 else 2_600_000), 64
    x = make(**sizes, seed=12)
    p = Plain(*x, window, **sizes)
    rows = torch.empty(S * ld, dtype=BF, device="cuda").view(S, ld)
    at = 0

    def place(t):
        nonlocal at
        at += t.shape[1] + 64
        place = rows[:, at - t.shape[1] - 64: at - 64]
        place.copy_(t)
        return place
    q, k, v, do = (place(x[i].cuda()) for i in (0, 1, 2, 4))
    lam = x[3].cuda()
    r = ops().diff_attn_fwd(q, k, v, lam, window=window, **sizes, out=place(torch.zeros(S, 2 * W)))
    check(r, p)
    grads = [place(torch.zeros(S, n * W)) for n in (2, 1, 1)]
    g = ops().diff_attn_bwd(q, k, v, lam, place(p.o.to(BF).cuda()), place(p.o2.to(BF).cuda()), p.lse.float().cuda(), do, window=window, **sizes, dq=grads[0], dk=grads[1], dv=grads[2])
    check_grads(g, p)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(g, grads))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,window", [(64, None), (32, None), (64, 40)])
def test_what_a_row_does_not_see_does_not_reach_it(D, window, value):
    """Infinities and NaN in one token's keys and values reach the queries that see it, in its query and dO the keys that it sees, and nothing else."""
    unseen(dict(B=2, S=200, H=4, KH=2, D=D), window, 100, value)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("D,window,S,at", [(64, None, 1700, 1500), (32, None, 4100, 70), (64, 1500, 2300, 700)])
def test_nor_where_chains_are_split(D, window, S, at, value):
    unseen(dict(B=1, S=S, H=2, KH=1, D=D), window, at, value)


@pytest.mark.parametrize("value", [math.nan, -math.inf])
@pytest.mark.parametrize("B,S,H,KH,D,window,at", [(41, 130, 16, 8, 64, None, 70), (41, 130, 16, 8, 32, 60, 3), (3, 300, 20, 20, 32, None, 128), (3, 300, 40, 20, 64, 33, 255)])
def test_nor_where_the_gpu_is_full(B, S, H, KH, D, window, at, value):
    unseen(dict(B=B, S=S, H=H, KH=KH, D=D), window, at, value)


def unseen(sizes, window, at, value):
    B, S, W = sizes["B"], sizes["S"], 2 * sizes["D"]
    T, last = B * S, min(S, at + window + 1) if window else S
    x = make(**sizes, seed=8)
    p = Plain(*x, window, **sizes)
    q, k, v, lam, do = (t.clone() for t in x)
    k[at, 1] = value
    v[at, 3] = value
    r = forward((q, k, v, lam, do), sizes, window)
    sees = torch.zeros(T, dtype=torch.bool)
    sees[at: last] = True
    rest = ~sees
    near(r.o[rest.cuda()], p.o[rest], p.o_room[rest], "o")
    near(r.o2[rest.cuda()], p.o2[rest], p.o2_room[rest], "o2")
    if sizes["KH"] > 1:
        near(r.o[:, 2 * W:], p.o[:, 2 * W:], p.o_room[:, 2 * W:], "the other group's heads")
    assert not r.o[at, : 2 * W].isfinite().all()
    lse = sees.view(B, S)
    keep = ~lse[:, None, None, :].expand_as(p.lse)
    near(r.lse[keep.cuda()], p.lse[keep], p.lse_room[keep], "lse")
    # dQ of the queries that do not see it; dK, dV of the keys that a bad query does not see
    g = backward((q, k, v, lam, do), p, sizes, window)
    near(g[0][rest.cuda()], p.grads[0][rest], p.dq_room[rest], "dq")
    q, k, v, lam, do = (t.clone() for t in x)
    q[at, 1] = value
    do[at, 2] = value
    g = backward((q, k, v, lam, do), p, sizes, window)
    seen = torch.zeros(T, dtype=torch.bool)
    seen[max(0, at - window) if window else 0: at + 1] = True
    for i, name in ((1, "dk"), (2, "dv")):
        near(g[i][~seen.cuda()], p.grads[i][~seen], getattr(p, name + "_room")[~seen], name)
    rest = torch.ones(T, dtype=torch.bool)
    rest[at] = False
    near(g[0][rest.cuda()], p.grads[0][rest], p.dq_room[rest], "dq of the other queries")


def test_a_longer_sequence():
    """2500 tokens: blocks of every kind, tiles in all rounds."""
    sizes = dict(B=1, S=2500, H=2, KH=1, D=64)
    x = make(**sizes, seed=9)
    for window in (None, 1000):
        p = Plain(*x, window, **sizes)
        check(forward(x, sizes, window), p)
        check_grads(backward(x, p, sizes, window), p)


def test_a_graph_replayed_over_new_inputs():
    """Forward and backward in one graph, replayed over changing inputs with eager work in between: the same bits as eager calls."""
    sizes = dict(B=2, S=190, H=4, KH=2, D=64)
    ins = [t.cuda() for t in make(**sizes, seed=0)]

    def step(q, k, v, lam, do):
        r = ops().diff_attn_fwd(q, k, v, lam, window=90, **sizes)
        return (r.o, r.lse, *ops().diff_attn_bwd(q, k, v, lam, r.o, r.o2, r.lse, do, window=90, **sizes))
    step(*ins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*ins)
    for rep in range(4):
        for a, b in zip(ins, make(**sizes, seed=20 + rep)):
            a.copy_(b)
        want = step(*ins)
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep


def test_two_graphs_share_a_pool():
    """Long chains, whose chunks lie in workspaces, in two graphs that take their memory from one pool, replayed in turn."""
    sizes = dict(B=1, S=1800, H=2, KH=1, D=64)
    works = [[t.cuda() for t in make(**sizes, seed=s)] for s in (1, 2)]

    def step(q, k, v, lam, do):
        r = ops().diff_attn_fwd(q, k, v, lam, **sizes)
        return (r.o, r.lse, *ops().diff_attn_bwd(q, k, v, lam, r.o, r.o2, r.lse, do, **sizes))
    want = [step(*w) for w in works]
    torch.cuda.synchronize()
    graphs, outs, pool = [torch.cuda.CUDAGraph() for _ in works], [], torch.cuda.graph_pool_handle()
    for g, w in zip(graphs, works):
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(*w))
    for rep in range(3):
        for i in (0, 1, 1, 0):
            for t in outs[i]:
                t.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i])), (rep, i)


@pytest.mark.parametrize("sizes", [dict(B=2, S=500, H=8, KH=2, D=64), dict(B=1, S=1800, H=2, KH=1, D=64)])
def test_two_streams_at_once(sizes):
    works = [[t.cuda() for t in make(**sizes, seed=s)] for s in (1, 2)]

    def step(q, k, v, lam, do):
        r = ops().diff_attn_fwd(q, k, v, lam, **sizes)
        return (r.o, r.lse, *ops().diff_attn_bwd(q, k, v, lam, r.o, r.o2, r.lse, do, **sizes))
    want = [step(*w) for w in works]
    streams = [torch.cuda.Stream() for _ in works]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (s, w) in enumerate(zip(streams, works)):
            with torch.cuda.stream(s):
                got[i] = step(*w)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals_of_the_wrappers():
    from olmax_amd._lib import OlmaxHipError
    sizes = dict(B=2, S=10, H=4, KH=2, D=64)
    q, k, v, lam, do = (t.cuda() for t in make(**sizes))
    r = ops().diff_attn_fwd(q, k, v, lam, **sizes)
    good = dict(q=q, k=k, v=v, lam=lam, o=r.o, o2=r.o2, lse=r.lse, do=do, **sizes)
    bad = [dict(q=q.float()), dict(k=k[:-1]), dict(v=v[:, :-8]), dict(lam=lam[:2]), dict(lam=lam.double()), dict(lam=lam.cpu()), dict(H=3), dict(D=128), dict(S=0), dict(KH=4), dict(q=q.t()),
           dict(v=torch.zeros(20, 264, dtype=BF, device="cuda")[:, 4:260]), dict(B=1)]
    for change in bad + [dict(o2=None), dict(o=r.o[:-1]), dict(lse=r.lse.view(-1)), dict(do=do.half()), dict(dq=q), dict(dk=r.o[:, :256]), dict(dv=v)]:
        with pytest.raises(OlmaxHipError):
            ops().diff_attn_bwd(**{**good, **change})
    for name in ("o", "o2", "lse", "do"):
        good.pop(name)
    for change in bad + [dict(out=q), dict(out=torch.zeros(20, 512, device="cuda"))]:
        with pytest.raises(OlmaxHipError):
            ops().diff_attn_fwd(**{**good, **change})


def test_a_block_of_them_all():
    """What a layer does: rotated queries and keys of a fused projection, the attention, and the gradients back through the rotation into the projection's rows, on a stream of
    its own, against the plain forms.  Bounds as above; each result is compared with what the plain form makes of the rounded numbers
    that go in."""
    B, S, H, KH, D = 2, 140, 4, 2, 64
    W, T = 2 * D, 280
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D)
    g = torch.Generator().manual_seed(11)
    base = torch.randn(T, (H + 2 * KH) * W, generator=g).to(BF)
    do, lam = torch.randn(T, H * W, generator=g).to(BF), torch.tensor([0.2, 0.4, 0.8, 0.6])
    p = torch.cat([torch.arange(100), torch.arange(40)]).repeat(B).to(torch.int32)
    heads = 2 * (H + KH)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cos, sin = ops().rotary_tables(4096, D, 5e5, "cuda", scaling=ops().RopeScaling("llama3", 8.0))
        qkv, lam_, do_, p_ = base.cuda(), lam.cuda(), do.cuda(), p.cuda()
        kw = dict(heads=heads, head_dim=D, positions=p_)
        ops().rotary_fwd(qkv, cos, sin, out=qkv, **kw)
        q, k, v = qkv.split([H * W, KH * W, KH * W], 1)
        r = ops().diff_attn_fwd(q, k, v, lam_, **sizes)
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = dqkv.split([H * W, KH * W, KH * W], 1)
        dlam = ops().diff_attn_bwd(q, k, v, lam_, r.o, r.o2, r.lse, do_, dq=dq, dk=dk, dv=dv, **sizes)[3]
        turned = dqkv.clone()
        ops().rotary_bwd(dqkv, cos, sin, out=dqkv, **kw)
    s.synchronize()
    c, sn = cos.cpu().double(), sin.cpu().double()
    want = base.double().clone()
    want[:, : heads * D] = ref.rotary(want[:, : heads * D], c, sn, p, heads=heads, head_dim=D)
    pairs = base.double().abs()[:, : heads * D].reshape(T, heads, 2, D // 2).sum(2, keepdim=True).expand(-1, -1, 2, -1).reshape(T, -1)
    room = want.abs() * H8
    room[:, : heads * D] += 3 * U * pairs
    near(qkv, want, room, "rotated")
    rounded = qkv.cpu()
    plain = Plain(*rounded.split([H * W, KH * W, KH * W], 1), lam, do, None, own=True, **sizes)
    check(r, plain)
    near(dlam, plain.grads[3], plain.dlam_room, "dlam")
    back = turned.cpu().double()
    for got, name, w in zip(back.split([H * W, KH * W, KH * W], 1), ("dq", "dk", "dv"), plain.grads):
        near(got, w, getattr(plain, name + "_room"), name)
    want = back.clone()
    want[:, : heads * D] = ref.rotary(back[:, : heads * D], c, sn, p, heads=heads, head_dim=D, back=True)
    pairs = back.abs()[:, : heads * D].reshape(T, heads, 2, D // 2).sum(2, keepdim=True).expand(-1, -1, 2, -1).reshape(T, -1)
    room = want.abs() * H8
    room[:, : heads * D] += 3 * U * pairs
    near(dqkv, want, room, "turned back")


@pytest.mark.parametrize("sizes,window", [(dict(B=1, S=200, H=4, KH=2, D=64), None), (dict(B=2, S=150, H=4, KH=2, D=32), 60), (dict(B=41, S=130, H=16, KH=8, D=64), None),
                                          (dict(B=1, S=1700, H=2, KH=1, D=64), None), (dict(B=1, S=4100, H=2, KH=1, D=32), None)])
def test_what_is_wrong_with_the_first_map_leaves_the_second_ones_results(sizes, window):
    """An infinity or NaN that only the first map or the weight has reaches o and the first map's log-normalisers; o2 and the second map's are the same bits as without it, whichever wave has stored
    them.  (Rows of o that do not see it may differ by roundings: a wave moves the reference of its exponentials for all of its rows.)  With a weight that is NaN nothing but its head's o changes."""
    H, D, S = sizes["H"], sizes["D"], sizes["S"]
    x = make(**sizes, seed=13)
    want = forward(x, sizes, window)
    at = 70
    last = min(S, at + window + 1) if window else S
    for name, value in (("q", math.inf), ("k", math.nan), ("k", -math.inf), ("lam", math.nan)):
        y = dict(zip(("q", "k", "v", "lam", "do"), (t.clone() for t in x)))
        if name == "lam":
            y["lam"][0] = value
        else:
            y[name][at, 1] = value  # (column 1 of a head: the first map's)
        r = forward(tuple(y.values()), sizes, window)
        assert torch.equal(r.o2, want.o2) and torch.equal(r.lse[:, :, 1], want.lse[:, :, 1]), name
        bad = torch.zeros(sizes["B"], S, dtype=torch.bool, device="cuda")
        bad[:1 if name != "lam" else None, at if name == "q" else at if name == "k" else 0: at + 1 if name == "q" else last if name == "k" else S] = True
        heads = slice(0, 1) if name != "k" else slice(0, H // sizes["KH"])
        o, clean = (t.view(-1, H, 2 * D) for t in (r.o, want.o))
        if value != -math.inf:  # (scores of minus infinity alone leave a row as it is)
            assert not o[bad.view(-1)][:, heads].isfinite().any(), name
        if name == "lam":
            assert torch.equal(o[:, 1:], clean[:, 1:]) and torch.equal(r.lse, want.lse)


def test_weights_between_the_rows_of_the_queries():
    """lam in the columns that a fused row has behind the queries: no operand's memory."""
    sizes = dict(B=2, S=90, H=4, KH=2, D=64)
    x = make(**sizes, seed=14)
    p = Plain(*x, None, **sizes)
    q, k, v, lam, do = (t.cuda() for t in x)
    wide = torch.zeros(180, 512 + 64, dtype=BF, device="cuda")
    wide[:, :512] = q
    for row in (0, 57, 179):
        between = wide[row, 512:520].view(torch.float32)
        between.copy_(lam)
        y = (wide[:, :512], k, v, between, do)
        r = ops().diff_attn_fwd(*y[:4], **sizes)
        check(r, p)
        check_grads(ops().diff_attn_bwd(*y[:4], p.o.to(BF).cuda(), p.o2.to(BF).cuda(), p.lse.float().cuda(), do, **sizes), p)


@pytest.mark.parametrize("sizes", [dict(B=1, S=300, H=8, KH=8, D=64), dict(B=41, S=130, H=16, KH=8, D=64), dict(B=2, S=1100, H=16, KH=8, D=64)])
@pytest.mark.parametrize("window", [0, 150])
def test_weights_gradient_at_large_scores(sizes, window):
    """Equal scores m, whole numbers that differ by head and go up to 1000, and dP = 64: every probability is one over the number of keys n that a row sees, and dlam is -64 times the number of rows (the
    log-normalisers are given, m + ln n rounded to fp32, and P = exp(m - that), which dlam is computed from here).  m's exponent is rounded by up to 2^-24 m log2(e), 9e-5 at 1000, which all of a
    head's rows share.  What is left: an exponential's 2^-23, three roundings of the row's factor and sum, the second order 2^-26 of that factor, at most 64 for n equal numbers, in
    tiles of 16, and for the rows', log2 (64 x rows) + 64 of u."""
    B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
    T = B * S
    g = torch.Generator().manual_seed(15)
    m = torch.randint(500, 1000, (KH,), generator=g).repeat_interleave(H // KH)
    # a score of m: q k / 8 with k = 8 in eight columns and q = m / 8 as a bf16 number above, and below, its lowest bits
    k = torch.zeros(T, KH, 2, D)
    k[..., :8] = 8.0
    q = torch.zeros(T, H, 2, D)
    q[..., 0] = (m - m % 8).float()[:, None]
    q[..., 1] = (m % 8).float()[:, None]
    v, do = torch.full((T, KH * 2 * D), 1.0), torch.zeros(T, H, 2 * D)
    do[..., 0] = 64.0
    lam = torch.linspace(0.1, 0.9, H)
    i = torch.arange(S)
    n = (torch.clamp(i, max=window) + 1).double()
    exact = m.double()[:, None] + n.log()[None, :]  # [H, S]
    lse = exact.float()
    p = torch.exp(m.double()[:, None] - lse.double())
    want = -64.0 * B * (p * n).sum(1)
    x = [t.reshape(T, -1).to(BF).cuda() for t in (q, k, v)]
    full = lse[None, :, None, :].expand(B, H, 2, S).contiguous().cuda()
    o = (torch.ones(T, H, 2 * D) * (1 - lam)[None, :, None]).reshape(T, -1).to(BF).cuda()
    got = ops().diff_attn_bwd(*x, lam.cuda(), o, torch.ones(T, H * 2 * D, dtype=BF, device="cuda"), full, do.reshape(T, -1).to(BF).cuda(), window=window, **sizes)[3]
    room = want.abs() * U * (2 + 3 + 1 + 64 + math.log2(64 * T) + 64)
    near(got, want, room, "dlam")


def test_a_workspace_that_is_not_needed_may_lie_anywhere():
    """Where the query returns 0 the workspace is no memory of the call's, whatever it points to."""
    from olmax_amd import _lib
    sizes = dict(B=2, S=90, H=4, KH=2, D=64)
    q, k, v, lam, _ = (t.cuda() for t in make(**sizes, seed=16))
    want = ops().diff_attn_fwd(q, k, v, lam, **sizes)
    assert ops()._size32("olmax_diff_attn_fwd_workspace_bytes", *sizes.values(), -1) == 0
    o, o2, lse = (torch.empty_like(t) for t in want)
    for at in (None, lse.data_ptr() + 64, o.data_ptr() + 64, q.data_ptr(), lam.data_ptr() + 4):
        _lib.check(_lib.typed("olmax_diff_attn_fwd")(_lib.raw_stream(), q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), o.data_ptr(), o2.data_ptr(), lse.data_ptr(), at, 0, *sizes.values(),
                                                     512, 256, 256, 512, 512, 0, -1))
        assert all(torch.equal(a, b) for a, b in zip((o, o2, lse), want))


@pytest.mark.parametrize("sizes,window", [(dict(B=1, S=1, H=4, KH=2, D=64), None), (dict(B=5, S=1, H=2, KH=1, D=32), 1024), (dict(B=700, S=1, H=8, KH=8, D=64), 0), (dict(B=2, S=2, H=8, KH=4, D=64), 0),
                                          (dict(B=1, S=200, H=4, KH=2, D=64), 0), (dict(B=1, S=333, H=4, KH=2, D=32), 0), (dict(B=41, S=130, H=16, KH=8, D=64), 0), (dict(B=2, S=1100, H=20, KH=10, D=32), 0),
                                          (dict(B=2, S=1100, H=16, KH=8, D=64), None), (dict(B=1, S=2111, H=1, KH=1, D=64), None), (dict(B=2, S=90, H=4, KH=2, D=32), 20)])
def test_a_query_that_sees_one_key_moves_nothing(sizes, window):
    """Its probabilities are 1 whatever queries and keys are: their gradients are exactly 0, not what roundings leave.  So they are where something that it does not see is not finite."""
    B, S = sizes["B"], sizes["S"]
    q, k, v, lam, do = (t.cuda() for t in make(**sizes, seed=17))
    r = ops().diff_attn_fwd(q, k, v, lam, window=window, **sizes)
    alone = torch.arange(S) == 0 if window != 0 else torch.ones(S, dtype=torch.bool)
    alone = alone.repeat(B).cuda()

    def grads(**changed):
        return ops().diff_attn_bwd(*(changed.get(n, t) for n, t in (("q", q), ("k", k), ("v", v))), lam, *r, changed.get("do", do), window=window, **sizes)
    g = grads()
    assert g[0][alone].eq(0).all() and (alone.all() or not g[0][~alone].eq(0).all(1).any())
    if alone.all():
        assert g[1].eq(0).all()
        assert torch.equal(g[2].eq(0).all(), torch.tensor(False, device="cuda"))
    if S > 5:
        k2, v2, q2, do2 = (t.clone() for t in (k, v, q, do))
        k2[5, 1] = v2[5, 3] = math.nan
        assert grads(k=k2, v=v2)[0][alone & (torch.arange(B * S, device="cuda") != 5)].eq(0).all()
        if window == 0:
            q2[5, 1] = do2[5, 2] = math.nan
            dk = grads(q=q2, do=do2)[1]
            assert dk[torch.arange(B * S, device="cuda") != 5].eq(0).all() and not dk[5].isfinite().all()
