"""Differential attention: what the entry points and their wrappers refuse.  No GPU needed: addresses are never read."""
import pytest

ARG, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -5


def lib():
    from olmax_amd import _lib
    if not _lib.lib_path().exists():
        pytest.skip("libolmax_hip.so not built")
    return _lib


def at(i):
    return (i + 1) << 28


B, S, H, KH, D = 2, 100, 4, 2, 64
Q, KV = H * 2 * D, KH * 2 * D
SIZES = dict(B=B, S=S, H=H, KH=KH, D=D)
FWD = dict(stream=None, q=at(0), k=at(1), v=at(2), lam=at(3), o=at(4), o2=at(5), lse=at(6), ws=at(12), nbytes=1 << 27, **SIZES, ldq=Q, ldk=KV, ldv=KV, ldo=Q, ldo2=Q, shared=0, window=-1)
BWD = dict(stream=None, q=at(0), k=at(1), v=at(2), lam=at(3), o=at(4), o2=at(5), lse=at(6), do=at(7), dq=at(8), dk=at(9), dv=at(10), dlam=at(11), ws=at(12), nbytes=1 << 27, **SIZES,
           ldq=Q, ldk=KV, ldv=KV, ldo=Q, ldo2=Q, lddo=Q, lddq=Q, lddk=KV, lddv=KV, shared=0, window=-1)
CALLS = {"olmax_diff_attn_fwd": FWD, "olmax_diff_attn_bwd": BWD}
BOTH = [(dict(B=0), SHAPE), (dict(S=0), SHAPE), (dict(S=(1 << 24) + 1), SHAPE), (dict(H=0), SHAPE), (dict(KH=0), SHAPE), (dict(KH=3), SHAPE), (dict(D=16), SHAPE), (dict(D=128), SHAPE),
        (dict(D=48), SHAPE), (dict(B=1 << 30), SHAPE)]
BOTH += [({p: None}, ARG) for p in ("q", "k", "v", "lam", "o", "lse")]
BOTH += [({p: at(0) + 8}, ALIGN) for p in ("q", "k", "v", "o", "o2")] + [({p: at(3) + 2}, ALIGN) for p in ("lam", "lse")]
BOTH += [({n: 4}, ALIGN) for n in ("ldq", "ldk", "ldv", "ldo", "ldo2")] + [({n: 1028}, ALIGN) for n in ("ldq", "ldk", "ldv", "ldo", "ldo2")] + [(dict(ldq=1 << 24), ALIGN), (dict(ldv=-512), ALIGN)]
ONLY_BWD = [({p: None}, ARG) for p in ("o2", "do", "dq", "dk", "dv", "dlam", "ws")] + [({p: at(20) + 8}, ALIGN) for p in ("do", "dq", "dk", "dv")]
ONLY_BWD += [(dict(dlam=at(11) + 1), ALIGN), (dict(nbytes=100), WORKSPACE), (dict(ws=at(12) + 16), WORKSPACE), (dict(lddk=128), ALIGN), (dict(lddo=516), ALIGN)]
# memory that an output shares with an input or another output
ONLY_BWD += [(dict(dq=at(0)), ARG), (dict(dk=at(1)), ARG), (dict(dq=at(7)), ARG), (dict(dv=at(9)), ARG), (dict(dk=at(9), dv=at(9) + 2 * KV, lddk=2 * KV, lddv=4 * KV), ARG),
             (dict(dk=at(8) + 2 * 128), ARG), (dict(dv=at(5) + 2 * Q * 3), ARG)]
FEW = dict(B=1, S=8192, H=1, KH=1)
ONLY_FWD = [({**FEW, "ws": None}, WORKSPACE), ({**FEW, "nbytes": 1000}, WORKSPACE), ({**FEW, "ws": at(12) + 8}, WORKSPACE), (dict(o=at(0)), ARG), (dict(o=at(2)), ARG), (dict(o2=at(4)), ARG), (dict(o2=at(4) + 2 * 64), ARG), (dict(o=at(1) - 2 * 64), ARG)]


@pytest.mark.parametrize("name,change,code", [(n, c, r) for n in CALLS for c, r in BOTH] + [("olmax_diff_attn_bwd", c, r) for c, r in ONLY_BWD] +
                         [("olmax_diff_attn_fwd", c, r) for c, r in ONLY_FWD])
def test_refuses(name, change, code):
    L = lib()
    assert set(change) <= set(CALLS[name])
    assert L.typed(name)(*{**CALLS[name], **change}.values()) == code, L.load().olmax_last_error_string()
    assert name.encode() in L.load().olmax_last_error_string()


def test_workspace_sizes():
    from olmax_amd import ops
    lib()
    size = lambda *a: ops._size32("olmax_diff_attn_bwd_workspace_bytes", *a)  # noqa: E731
    assert size(0, 1, 1, 1, 64, -1) == size(1, 0, 1, 1, 64, -1) == size(1, 1, 0, 1, 64, -1) == size(1, 1, 1, 0, 64, -1) == size(1, 1, 1, 1, 48, -1) == 0
    assert size(1, 1, 1, 1, 64, -1) > 0
    assert size(8, 1 << 20, 128, 32, 64, -1) > 1 << 32  # (beyond 32 bits)
    size = lambda *a: ops._size32("olmax_diff_attn_fwd_workspace_bytes", *a)  # noqa: E731
    assert size(0, 8192, 1, 1, 64, -1) == size(1, 8192, 1, 1, 48, -1) == size(1, 100, 4, 2, 64, -1) == size(2, 4096, 32, 8, 64, -1) == 0
    assert size(1, 8192, 1, 1, 64, -1) > 8192 * 2 * (256 + 4) * 4 - 1  # a long sequence of one head is split


def test_wrappers_refuse():
    import torch

    from olmax_amd import ops
    from olmax_amd._lib import OlmaxHipError
    q, lam = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(1)
    with pytest.raises(OlmaxHipError):
        ops.diff_attn_fwd(q, q, q, lam, B=1, S=4, H=1, KH=1, D=32)
    with pytest.raises(OlmaxHipError):
        ops.diff_attn_bwd(q, q, q, lam, q, q, lam, q, B=1, S=4, H=1, KH=1, D=32)


@pytest.mark.parametrize("window", [None, 0, 3])
@pytest.mark.parametrize("shared", [False, True])
def test_gradients_of_the_plain_form_are_autograds_and_the_differences(window, shared):
    """float64 through some 30 operations: 1e-12; central differences: h^2 of the third derivative, 2^-52 / h of a sum of 200 numbers."""
    import torch

    from oracle import ref
    g = torch.Generator().manual_seed(1)
    sizes = dict(B=2, S=9, H=4, KH=2, D=4)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)  # noqa: E731
    ins = [mk(18, 32), mk(18, 16), mk(18, 16), mk(1 if shared else 4)]
    do = torch.randn(18, 32, generator=g, dtype=torch.float64)
    f = lambda *a: (ref.diff_attn_fwd(*a, **sizes, window=window)[0] * do).sum()  # noqa: E731
    want = torch.autograd.grad(f(*ins), ins)
    ins = [t.detach() for t in ins]
    got = ref.diff_attn_bwd(*ins, do, **sizes, window=window)
    for a, b, t in zip(got, want, range(4)):
        assert a.shape == ins[t].shape and (a - b).abs().max() < 1e-12
        for at in (0, ins[t].numel() // 2, ins[t].numel() - 1):
            up, down = [x.clone() for x in ins], [x.clone() for x in ins]
            up[t].view(-1)[at] += 1e-5
            down[t].view(-1)[at] -= 1e-5
            assert abs((f(*up) - f(*down)) / 2e-5 - a.reshape(-1)[at]) < 1e-8


def test_plain_form_is_two_attentions():
    import torch

    from oracle import ref
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(7, n, generator=g, dtype=torch.float64) for n in (16, 16, 16))
    lam = torch.tensor([0.3, -1.5], dtype=torch.float64)
    o, o2, lse = ref.diff_attn_fwd(q, k, v, lam, B=1, S=7, H=2, KH=2, D=4)
    for h in range(2):
        m = [torch.nn.functional.scaled_dot_product_attention(q[None, :, h * 8 + x: h * 8 + x + 4], k[None, :, h * 8 + x: h * 8 + x + 4], v[None, :, h * 8: h * 8 + 8], is_causal=True)[0]
             for x in (0, 4)]
        assert (o[:, h * 8: h * 8 + 8] - (m[0] - lam[h] * m[1])).abs().max() < 1e-12 and (o2[:, h * 8: h * 8 + 8] - m[1]).abs().max() < 1e-12
        assert abs(lse[0, h, 1, 0] - (q[0, h * 8 + 4: h * 8 + 8] * k[0, h * 8 + 4: h * 8 + 8]).sum() / 2) < 1e-12


ONE_ROW = dict(S=1, KH=64, H=64)


@pytest.mark.parametrize("name,change,code", [  # 2^32 threads and more; one workgroup's fewer pass on to what is refused next
    ("olmax_diff_attn_fwd", dict(B=1 << 17, D=64, **ONE_ROW), SHAPE), ("olmax_diff_attn_fwd", dict(B=(1 << 17) - 1, D=64, **ONE_ROW), ALIGN),
    ("olmax_diff_attn_fwd", dict(B=1 << 18, D=32, **ONE_ROW), SHAPE), ("olmax_diff_attn_fwd", dict(B=(1 << 18) - 1, D=32, **ONE_ROW), ALIGN),
    ("olmax_diff_attn_bwd", dict(B=1 << 18, D=64, **ONE_ROW), SHAPE), ("olmax_diff_attn_bwd", dict(B=(1 << 18) - 1, D=64, **ONE_ROW), ALIGN),
    ("olmax_diff_attn_bwd", dict(B=1 << 18, D=32, **ONE_ROW), SHAPE), ("olmax_diff_attn_bwd", dict(B=(1 << 18) - 1, D=32, **ONE_ROW), ALIGN),
    ("olmax_diff_attn_fwd", dict(B=1 << 6, S=1 << 24, H=1, KH=1, D=64), SHAPE), ("olmax_diff_attn_fwd", dict(B=(1 << 6) - 1, S=1 << 24, H=1, KH=1, D=64), ALIGN),
    ("olmax_diff_attn_fwd", dict(B=(1 << 31) - 1, S=1 << 24, H=1 << 16, KH=1 << 16), SHAPE), ("olmax_diff_attn_bwd", dict(B=(1 << 31) - 1, S=1 << 24, H=1 << 16, KH=1 << 16), SHAPE)])
def test_refuses_more_workgroups_than_a_launch_takes(name, change, code):
    L = lib()
    assert L.typed(name)(*{**CALLS[name], **change, "q": at(0) + 8}.values()) == code, L.load().olmax_last_error_string()


WIDE = dict(ldq=Q + 64, ldk=Q + 64, ldv=Q + 64)  # rows of a wider buffer: room for 64 numbers behind each
LAST = 2 * (B * S - 1)  # bytes to the last row of a stride of 1


@pytest.mark.parametrize("name,change,code", [
    ("olmax_diff_attn_fwd", dict(lse=at(0)), ARG), ("olmax_diff_attn_fwd", dict(lse=at(1) + LAST * KV + 2 * KV - 4), ARG), ("olmax_diff_attn_fwd", dict(lse=at(2) - 4 * B * H * 2 * S + 4), ARG),
    ("olmax_diff_attn_fwd", dict(lse=at(4) + 1024), ARG), ("olmax_diff_attn_fwd", dict(lse=at(5) + 1024), ARG), ("olmax_diff_attn_fwd", dict(lse=at(3) - 8), ARG),
    ("olmax_diff_attn_fwd", dict(lam=at(4) + 2 * Q), ARG), ("olmax_diff_attn_fwd", dict(lam=at(5) + 4, shared=1), ARG),
    ("olmax_diff_attn_fwd", dict(lse=at(0) + 2 * Q, **WIDE), ARG), ("olmax_diff_attn_fwd", dict(lam=at(4) + 2 * Q - 4, ldo=Q + 64), ARG),
    ("olmax_diff_attn_fwd", dict(lam=at(6) + 4 * B * H * 2 * S - 4, shared=1), ARG),
    ("olmax_diff_attn_bwd", dict(dlam=at(3)), ARG), ("olmax_diff_attn_bwd", dict(dlam=at(3) + 12), ARG), ("olmax_diff_attn_bwd", dict(dlam=at(6) + 64), ARG), ("olmax_diff_attn_bwd", dict(dlam=at(8)), ARG),
    ("olmax_diff_attn_bwd", dict(dlam=at(0) + 256), ARG), ("olmax_diff_attn_bwd", dict(dlam=at(12) + 1024), ARG), ("olmax_diff_attn_bwd", dict(ws=at(7)), ARG), ("olmax_diff_attn_bwd", dict(ws=at(10) - 256), ARG),
    ("olmax_diff_attn_bwd", dict(ws=at(6)), ARG), ("olmax_diff_attn_bwd", dict(lse=at(9) + 4), ARG), ("olmax_diff_attn_bwd", dict(lam=at(8) + LAST * Q), ARG)])
def test_refuses_memory_that_log_normalisers_weights_and_workspaces_share(name, change, code):
    L = lib()
    assert L.typed(name)(*{**CALLS[name], **change}.values()) == code and b"share" in L.load().olmax_last_error_string()


@pytest.mark.parametrize("change", [dict(ws=at(0)), dict(ws=at(4)), dict(ws=at(6)), dict(ws=at(3) - 64), dict(ws=at(2) - 64)])
def test_refuses_a_forward_workspace_in_other_memory(change):
    L = lib()
    few = {**FWD, **FEW, **{n: 2 * 64 for n in ("ldq", "ldk", "ldv", "ldo", "ldo2")}}
    assert L.typed("olmax_diff_attn_fwd")(*{**few, **change}.values()) == ARG and b"share" in L.load().olmax_last_error_string()
