"""GPU parity tests of differential attention's forms on large grids and long sequences, against the plain form in 64 bits.

A call runs with all of its heads, and some of its key heads are compared, with the bounds of test_diff_attn_gpu.py."""
import math

import pytest
import torch

from oracle import ref
from test_diff_attn_gpu import BF, H8, U, Plain, check, make, near, ops

pytestmark = pytest.mark.gpu


def group_of(t, g, sizes):
    """The columns of key head g, or of its query heads."""
    n, rep = 2 * sizes["D"], sizes["H"] // sizes["KH"]
    n *= rep if t.shape[1] == 2 * sizes["D"] * sizes["H"] else 1
    return t[:, g * n: (g + 1) * n]


def part_of(x, g, sizes):
    """A call with key head g alone."""
    rep = sizes["H"] // sizes["KH"]
    q, k, v, lam, do = x
    cut = lambda t: group_of(t, g, sizes) if sizes["KH"] > 1 else t  # noqa: E731
    return (cut(q), cut(k), cut(v), lam if lam.shape[0] != sizes["H"] else lam[g * rep: (g + 1) * rep], cut(do)), {**sizes, "H": rep, "KH": 1}


def run_and_compare(sizes, window, groups, lam=None, seed=0, dq_room=None):
    B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
    rep = H // KH
    x = list(make(**sizes, seed=seed))
    if lam is not None:
        x[3] = lam
    q, k, v, w, do = (t.cuda() for t in x)
    r = ops().diff_attn_fwd(q, k, v, w, window=window, **sizes)
    plains = {}
    o, o2, lse = r.o.clone(), r.o2.clone(), r.lse.clone()
    for g in groups:
        part, small = part_of(x, g, sizes)
        plains[g] = p = Plain(*part, window, **small)
        heads = slice(g * rep, (g + 1) * rep)
        near(r.lse[:, heads], p.lse, p.lse_room, f"lse of {g}")
        for got, name in ((r.o, "o"), (r.o2, "o2")):
            near(got.view(B * S, H, 2 * D)[:, heads].reshape(B * S, -1), getattr(p, name), getattr(p, name + "_room"), f"{name} of {g}")
        o.view(B * S, H, 2 * D)[:, heads] = p.o.to(BF).cuda().view(B * S, rep, 2 * D)
        o2.view(B * S, H, 2 * D)[:, heads] = p.o2.to(BF).cuda().view(B * S, rep, 2 * D)
        lse[:, heads] = p.lse.float().cuda()
    grads = ops().diff_attn_bwd(q, k, v, w, o, o2, lse, do, window=window, **sizes)
    for g in groups:
        p, heads = plains[g], slice(g * rep, (g + 1) * rep)
        part, small = part_of(x, g, sizes)
        dq, dk, dv = (t.view(B * S, -1, 2 * D) for t in grads[:3])
        near(dq[:, heads].reshape(B * S, -1), p.grads[0], p.dq_room if dq_room is None else dq_room(part, p, window, small), f"dq of {g}")
        near(dk[:, g], p.grads[1], p.dk_room, f"dk of {g}")
        near(dv[:, g], p.grads[2], p.dv_room, f"dv of {g}")
        if w.shape[0] == H:
            near(grads[3][heads], p.grads[3].view(-1), p.dlam_room.view(-1), f"dlam of {g}")
    assert all(t.isfinite().all() for t in (*r, *grads))


def dq_room_of_own_sums(x, p, window, sizes):
    """Bound of dq whose delta is the kernel's own sum of P dP (see Plain): nothing in it is the weight's but the second map's factor."""
    B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
    q, k, v, lam, do = (t.double() for t in x)
    s, seen, _, kh = ref._diff_maps(q, k, B, S, H, KH, D, window)
    pr = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    A = ref._diff_maps(q.abs(), k.abs(), B, S, H, KH, D, window)[0].masked_fill(~seen, 0.0).amax(-1)
    e = (U * (D + 16 + (D + 12) * A + 4 * math.log(S + 1) + 2 * p.lse.abs()))[..., None]
    v_ = v.reshape(B, S, KH, 2 * D).permute(0, 2, 1, 3).repeat_interleave(H // KH, 1)
    do_ = do.reshape(B, S, H, 2 * D).permute(0, 2, 1, 3)
    dp, big = (do_ @ v_.transpose(-1, -2))[:, :, None], (do_.abs() @ v_.abs().transpose(-1, -2))[:, :, None]
    ds = (pr * (dp - (pr * dp).sum(-1, keepdim=True))).abs()
    off = (pr * big).sum(-1, keepdim=True) * (e + (2 * D + S) * U)
    room = (H8 + 2 * e) * ds + pr * (off + 2 * D * U * big) * (1 + H8) + S * U * ds
    w = lam.expand(H).abs()[:, None, None]
    room = room * torch.stack([torch.ones_like(w), w], 1) * D ** -0.5
    return (room @ kh.abs()).permute(0, 3, 1, 2, 4).reshape(B * S, -1) + H8 * p.grads[0].abs() + 1e-30


@pytest.mark.parametrize("sizes,window", [(dict(B=2, S=1100, H=16, KH=8, D=64), None), (dict(B=2, S=1100, H=20, KH=10, D=32), 700), (dict(B=1, S=2111, H=1, KH=1, D=64), None),
                                          (dict(B=1, S=1700, H=4, KH=4, D=64), None), (dict(B=1, S=3000, H=2, KH=1, D=32), 2500)])
@pytest.mark.parametrize("weight", [30.0, -4.0, 1.25])
def test_large_weights_leave_the_first_maps_gradient_exact(sizes, window, weight):
    """dq of long rows with weights above 1: its bound does not grow with them."""
    lam = torch.full((sizes["H"],), weight)
    run_and_compare(sizes, window, [0, sizes["KH"] - 1], lam=lam, seed=21, dq_room=dq_room_of_own_sums)


def test_a_large_weight_beside_small_ones():
    sizes = dict(B=2, S=1100, H=16, KH=8, D=64)
    lam = torch.tensor([0.5, -30.0] * 8)
    run_and_compare(sizes, None, [3], lam=lam, seed=22)
    run_and_compare({**sizes, "H": 1, "KH": 1}, None, [0], lam=torch.tensor([30.0]), seed=23, dq_room=dq_room_of_own_sums)


# olmax_diff_attn_form's bits
FWD64, FWD_DEALT, DQ_SPLIT, DQ_DEALT, LONG, KV4, KV8, KV_DEALT = (1 << i for i in range(8))
FORMS = [  # B, S, H, KH, D, window, form, weights shared, key heads that are compared
    (2, 1100, 40, 40, 64, None, LONG, False, (0, 39)), (2, 1100, 40, 40, 64, 700, LONG, True, (7, 39)), (2, 1100, 80, 40, 64, None, LONG, False, (0, 20)),
    (2, 1100, 16, 8, 64, None, LONG | KV4, False, (0, 7)), (2, 1100, 16, 8, 64, 600, LONG | KV4, False, (0, 7)), (2, 1300, 24, 12, 64, 900, LONG | KV4, True, (11,)),
    (1, 3000, 32, 8, 64, None, LONG | KV_DEALT, False, (5,)), (1, 4001, 32, 16, 64, 1024, LONG | KV4, False, (9,)),
    (2, 1100, 16, 16, 32, None, FWD64 | LONG | KV4, False, (0, 15)), (2, 1100, 32, 16, 32, None, FWD64 | LONG | KV4, False, (0, 15)), (1, 1500, 24, 12, 32, 400, LONG | FWD64 | KV4, False, (3,)),
    (2, 1100, 48, 12, 32, None, FWD64 | LONG | KV4, True, (0,)), (2, 1100, 40, 40, 32, None, FWD64 | LONG, False, (0, 39)), (2, 1100, 80, 40, 32, 700, FWD64 | LONG, False, (13,)),
    (1, 1100, 4, 4, 64, 700, DQ_SPLIT | FWD64 | LONG | KV4, False, (0, 3)), (1, 1300, 16, 2, 32, 900, FWD64 | DQ_SPLIT | LONG | KV_DEALT, False, (1,)),
    (1, 4000, 8, 2, 64, 1024, DQ_SPLIT | LONG | KV_DEALT, False, (0,)), (1, 4000, 8, 2, 32, 1024, FWD64 | DQ_SPLIT | LONG | KV8, False, (0,))]


@pytest.mark.parametrize("B,S,H,KH,D,window,form,shared,groups", FORMS)
def test_forms_of_large_grids_and_long_sequences(B, S, H, KH, D, window, form, shared, groups):
    print(f"[case] diff B{B} S{S} H{H} KH{KH} D{D} w{window} form{form}", flush=True)
    lam = torch.full((1,), 0.7) if shared else torch.rand(H, generator=torch.Generator().manual_seed(S)) * 1.2 - 0.3
    run_and_compare(dict(B=B, S=S, H=H, KH=KH, D=D), window, groups, lam=lam, seed=S + H)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("sizes,window,at", [(dict(B=2, S=1100, H=16, KH=8, D=64), None, 800), (dict(B=2, S=1100, H=40, KH=20, D=32), 700, 90), (dict(B=2, S=1100, H=40, KH=40, D=64), None, 1000)])
def test_what_a_row_does_not_see_does_not_reach_it_in_long_rows(sizes, window, at, value):
    """As test_what_a_row_does_not_see_does_not_reach_it, in the forms of large grids."""
    B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
    T, rep, W, last = B * S, H // KH, 2 * D, min(S, at + window + 1) if window else S
    x = make(**sizes, seed=31)
    part, small = part_of(x, 0, sizes)
    p = Plain(*part, window, **small)

    def backward(**changed):
        q, k, v, lam, do = (changed.get(n, t).cuda() for n, t in zip(("q", "k", "v", "lam", "do"), x))
        r = ops().diff_attn_fwd(q, k, v, lam, window=window, **sizes)
        o, o2, lse = r.o.clone(), r.o2.clone(), r.lse.clone()
        o[:, : rep * W], o2[:, : rep * W], lse[:, :rep] = p.o.to(BF).cuda(), p.o2.to(BF).cuda(), p.lse.float().cuda()
        return r, ops().diff_attn_bwd(q, k, v, lam, o, o2, lse, do, window=window, **sizes)
    k, v = x[1].clone(), x[2].clone()
    k[at, 1] = v[at, 3] = value
    r, g = backward(k=k, v=v)
    rest = torch.ones(T, dtype=torch.bool)
    rest[at: last] = False
    for got, name in ((r.o, "o"), (r.o2, "o2"), (g[0], "dq")):
        want = getattr(p, name) if name != "dq" else p.grads[0]
        near(got[rest.cuda()][:, : rep * W], want[rest], getattr(p, name + "_room")[rest], name)
    assert not r.o[at: last, : rep * W].isfinite().all(1).any() and r.o[:, rep * W:].isfinite().all()
    q, do = x[0].clone(), x[4].clone()
    q[at, 1] = do[at, 2] = value
    _, g = backward(q=q, do=do)
    rest = torch.ones(T, dtype=torch.bool)
    rest[max(0, at - window) if window else 0: at + 1] = False
    for i, name in ((1, "dk"), (2, "dv")):
        near(g[i][rest.cuda()][:, :W], p.grads[i][rest], getattr(p, name + "_room")[rest], name)
    rest = torch.ones(T, dtype=torch.bool)
    rest[at] = False
    near(g[0][rest.cuda()][:, : rep * W], p.grads[0][rest], p.dq_room[rest], "dq of the other queries")
