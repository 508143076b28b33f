"""GPU parity tests of rotary tables and rotations against the plain forms in 64 bits.

Tolerances, u = 2^-24.  Tables: an angle's fraction of a turn is exact to 2^-52 of its turns (below 2^18 here), the rest of a quarter turn is rounded once (at most pi/4), its polynomial in five
steps, whose lowest adds 1 u of the result and the others less together, and times the size once: 4 u of the size, 6 are allowed.  Rotations: two products and a sum in fp32, the first product rounded, then the sum: 2 u
of |a| + |b| times the table's largest entry, and the type's half step on the result (fp32's is in 3 u).  Columns that pass are the same bits."""
import math

import pytest
import torch

from oracle import ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def ops():
    from olmax_amd import ops
    return ops


SCALINGS = [(None, {}), ("linear", dict(factor=4.0)), ("llama3", dict(factor=8.0)), ("llama3", dict(factor=2.0, original_length=4096, low_turns=2.0, high_turns=9.0)),
            ("yarn", dict(factor=4.0, original_length=4096)), ("yarn", dict(factor=16.0, attention_factor=1.0, low_turns=0.5, high_turns=64.0)), ("yarn", dict(factor=2.0, original_length=3))]


@pytest.mark.parametrize("kind,more", SCALINGS)
@pytest.mark.parametrize("length,rotary,theta", [(1, 2, 1e4), (300, 64, 1e4), (131072, 128, 5e5), (77, 512, 1e6), (1000, 6, 1.5), (4097, 100, 5e5)])
def test_tables(kind, more, length, rotary, theta):
    scaling = None if kind is None else ops().RopeScaling(kind, **more)
    cos, sin = ops().rotary_tables(length, rotary, theta, "cuda", scaling=scaling)
    kw, size = {}, 1.0
    if kind is not None:
        _, factor, original, low, high, size = scaling.c_args()
        kw = dict(kind=kind, factor=factor, original_length=original, low_turns=low, high_turns=high)
        size = float(torch.tensor(size, dtype=F32))
    rows = torch.arange(length) if length < 5000 else torch.cat([torch.arange(100), torch.arange(length - 100, length), torch.randint(0, length, (500,), generator=torch.Generator().manual_seed(1))])
    angle = rows.double()[:, None] * ref.rotary_freqs(rotary, theta, **kw)
    assert cos.shape == sin.shape == (length, rotary // 2)
    assert (cos.cpu().double()[rows] - size * angle.cos()).abs().max() <= 6 * U * size
    assert (sin.cpu().double()[rows] - size * angle.sin()).abs().max() <= 6 * U * size
    assert cos[0].eq(size).all() and sin[0].eq(0).all()


def tables(rows, half, seed=3):
    """Any numbers do as tables: of both signs, up to 1.3."""
    t = torch.rand(2, rows, half, generator=torch.Generator().manual_seed(seed)) * 2.6 - 1.3
    return t[0].cuda(), t[1].cuda()


def check(y, x, cos, sin, p, heads, head_dim, layout, back):
    x64 = x[:, : heads * head_dim].cpu().double()
    want = ref.rotary(x64, cos.cpu().double(), sin.cpu().double(), p.cpu(), heads=heads, head_dim=head_dim, layout=layout, back=back)
    got = y[:, : heads * head_dim].cpu().double()
    T, R = x.shape[0], 2 * cos.shape[1]
    h = x64.view(T, heads, head_dim)
    a, b = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    room = torch.zeros_like(h)
    room[..., a] = room[..., b] = (h[..., a].abs() + h[..., b].abs()) * 1.3 * (3 * U)
    bound = room.view(T, -1) + (want.abs() * torch.finfo(BF).eps / 2 * (1 + 2 ** -10) if x.dtype == BF else 0.0)
    assert torch.equal(got.isnan(), want.isnan())
    assert (((got - want).abs() <= bound) | want.isnan()).all()
    left = torch.ones(head_dim, dtype=torch.bool)
    left[:R] = False
    assert torch.equal(got.view(T, heads, head_dim)[..., left], h[..., left])
    assert torch.equal(got[p.cpu() < 0], x64[p.cpu() < 0])


SHAPES = [  # tokens, heads, head_dim, rotary_dim
    (1, 1, 2, 2), (1, 40, 128, 128), (3, 5, 128, 128), (257, 12, 64, 64), (100, 9, 128, 32), (50, 7, 80, 16), (33, 3, 96, 96), (20, 4, 24, 20), (11, 3, 7, 4), (40, 130, 64, 32), (9, 2, 512, 512),
    (5, 1, 4096, 64), (64, 300, 16, 16), (1000, 1, 128, 64)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,head_dim,rotary", SHAPES)
def test_rotation(tokens, heads, head_dim, rotary, layout, dtype):
    g = torch.Generator().manual_seed(tokens + head_dim)
    x = torch.randn(tokens, heads * head_dim, generator=g).to(dtype).cuda()
    cos, sin = tables(60, rotary // 2)
    for back, call in ((False, ops().rotary_fwd), (True, ops().rotary_bwd)):
        y = call(x, cos, sin, heads=heads, head_dim=head_dim, seq_len=37, layout=layout)
        check(y, x, cos, sin, torch.arange(tokens) % 37, heads, head_dim, layout, back)
    p = torch.randint(-2, 60, (tokens,), generator=g).to(torch.int32)
    y = ops().rotary_fwd(x, cos, sin, heads=heads, head_dim=head_dim, positions=p.cuda(), layout=layout)
    check(y, x, cos, sin, p, heads, head_dim, layout, False)
    # in place, and the same bits
    z = x.clone()
    assert ops().rotary_fwd(z, cos, sin, heads=heads, head_dim=head_dim, positions=p.cuda(), layout=layout, out=z) is z
    assert torch.equal(z, y)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset,stride,ostride", [(0, 1536, 1024), (64, 1280, 1032), (1, 1100, 1027), (8, 1288, 1025)])
def test_views_of_wider_rows(offset, stride, ostride, layout, dtype):
    """Queries and keys in the rows of a fused projection, at any alignment; what is not theirs stays."""
    T, heads, D = 50, 8, 128
    g = torch.Generator().manual_seed(4)
    base = torch.randn(T, stride, generator=g).to(dtype).cuda()
    x = base[:, offset: offset + heads * D]
    cos, sin = tables(T, 32)
    full = torch.full((T, ostride), 7.0, dtype=dtype, device="cuda")
    y = ops().rotary_fwd(x, cos, sin, heads=heads, head_dim=D, layout=layout, out=full[:, : heads * D] if ostride == 1024 else full)
    check(y, x, cos, sin, torch.arange(T), heads, D, layout, False)
    assert full[:, heads * D:].eq(7.0).all()
    before = base.clone()
    ops().rotary_fwd(x, cos, sin, heads=heads, head_dim=D, layout=layout, out=x)
    assert torch.equal(x, y[:, : heads * D])
    assert torch.equal(base[:, :offset], before[:, :offset]) and torch.equal(base[:, offset + heads * D:], before[:, offset + heads * D:])


def test_positions_beyond_the_tables_show():
    x = torch.randn(6, 128, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    cos, sin = tables(10, 16)
    p = torch.tensor([0, 9, 10, 2 ** 31 - 1, -1, -2 ** 31], dtype=torch.int32)
    for layout in ("half", "interleaved"):
        y = ops().rotary_fwd(x, cos, sin, heads=2, head_dim=64, positions=p.cuda(), layout=layout)
        check(y, x, cos, sin, p, 2, 64, layout, False)
        assert y[2:4].view(2, 2, 64)[..., :32].isnan().all() and not y[[0, 1, 4, 5]].isnan().any()


def test_infinities_stay_in_their_pair():
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(0)).to(BF)
    x[1, 3], x[2, 130] = math.inf, math.nan
    x = x.cuda()
    cos, sin = tables(4, 32)
    y = ops().rotary_fwd(x, cos, sin, heads=2, head_dim=128)
    bad = ~y.isfinite()
    assert bad.sum() == 4 and bad[1, [3, 35]].all() and bad[2, [130, 162]].all()


def test_far_rows():
    """Rows whose offsets pass 32 bits: 9 of them, 2^28 elements apart."""
    T, heads, D = 9, 2, 64
    base = torch.empty(8 * 2 ** 28 + heads * D, dtype=BF, device="cuda")
    x = base.as_strided((T, heads * D), (2 ** 28, 1))
    x.copy_(torch.randn(T, heads * D, generator=torch.Generator().manual_seed(0)).to(BF))
    cos, sin = tables(T, 32)
    for layout in ("half", "interleaved"):
        y = ops().rotary_fwd(x, cos, sin, heads=heads, head_dim=D, layout=layout)
        check(y, x, cos, sin, torch.arange(T), heads, D, layout, False)


def test_refusals_of_the_wrappers():
    from olmax_amd._lib import OlmaxHipError
    x = torch.zeros(4, 128, dtype=BF, device="cuda")
    cos, sin = tables(4, 32)
    good = dict(heads=2, head_dim=64)
    for bad in (dict(x=x.half()), dict(x=x[:, ::2]), dict(x=x[0]), dict(cos=cos.double()), dict(cos=cos[:, :16]), dict(cos=cos.t().contiguous().t()), dict(sin=sin.cpu()),
                dict(positions=torch.zeros(4, device="cuda")), dict(positions=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(positions=torch.zeros(4, dtype=torch.int64, device="cuda")),
                dict(layout="pairs"), dict(heads=3), dict(heads=0), dict(seq_len=5), dict(seq_len=0), dict(out=torch.zeros(4, 128, device="cuda")), dict(out=x[:, 2:]), dict(head_dim=32, heads=4)):
        a = {**dict(x=x, cos=cos, sin=sin, **good), **bad}
        with pytest.raises(OlmaxHipError):
            ops().rotary_fwd(a.pop("x"), a.pop("cos"), a.pop("sin"), **a)
    for bad in (dict(length=0), dict(rotary_dim=5), dict(theta=0.5)):
        with pytest.raises(OlmaxHipError):
            ops().rotary_tables(**{**dict(length=4, rotary_dim=4, theta=1e4, device="cuda"), **bad})
    with pytest.raises(OlmaxHipError):
        ops().rotary_tables(4, 4, 1e4, "cuda", scaling=ops().RopeScaling("linear", 0.5))


def test_no_tokens():
    cos, sin = tables(4, 32)
    assert ops().rotary_fwd(torch.zeros(0, 128, dtype=BF, device="cuda"), cos, sin, heads=2, head_dim=64).shape == (0, 128)


def test_a_graph_replayed_over_new_rows():
    T, heads, D = 70, 6, 64
    cos, sin = tables(100, 32)
    x, p = torch.zeros(T, heads * D, dtype=BF, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    kw = dict(heads=heads, head_dim=D, positions=p, layout="interleaved")
    ops().rotary_fwd(x, cos, sin, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops().rotary_fwd(x, cos, sin, **kw)
        ops().rotary_bwd(y, cos, sin, out=y, **kw)
    for rep in range(4):
        g = torch.Generator().manual_seed(rep)
        x.copy_(torch.randn(T, heads * D, generator=g).to(BF))
        p.copy_(torch.randint(-1, 100, (T,), generator=g))
        want = ops().rotary_bwd(ops().rotary_fwd(x, cos, sin, **kw), cos, sin, **kw)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), rep


def test_another_stream():
    x = torch.randn(300, 512, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    cos, sin = tables(300, 32)
    want = ops().rotary_fwd(x, cos, sin, heads=8, head_dim=64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops().rotary_fwd(x, cos, sin, heads=8, head_dim=64)
    s.synchronize()
    assert torch.equal(got, want)


def test_agrees_with_the_half_rotation_of_whole_heads():
    """qk_rope_fwd computes the same products in another order: both are within a half step of bf16 and 3 u of the two products."""
    T, heads, D = 130, 4, 128
    x = torch.randn(T, heads * D, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    cos, sin = ops().rope_tables(65, D, 1e4, "cuda")
    a, b = ops().qk_rope_fwd(x, cos, sin, heads=heads, head_dim=D, seq_len=65), ops().rotary_fwd(x, cos, sin, heads=heads, head_dim=D)
    room = torch.maximum(a.double().abs(), b.double().abs()) * torch.finfo(BF).eps + 16 * 6 * U
    assert ((a.double() - b.double()).abs() <= room).all()


def _scaled(scaling):
    """The oracle's table function with a layer's scaling; `scaling` by theta."""
    def tables(S, D, theta, dtype=torch.float32):
        c = scaling[theta]
        kw = {} if c is None else dict(kind=c.kind, factor=c.factor, original_length=c.original_length, low_turns=c.low_turns, high_turns=c.c_args()[4])
        angle = torch.arange(S, dtype=torch.float64)[:, None] * ref.rotary_freqs(D, theta, **kw)
        size = 1.0 if c is None else c.c_args()[5]
        return (size * angle.cos()).to(dtype), (size * angle.sin()).to(dtype)
    return tables


@pytest.mark.parametrize("kind,scalings", [("default", ("yarn", "yarn")), ("reordered_norm", ("yarn", None)), ("reordered_norm", ("llama3", "linear"))])
def test_a_model_with_scaled_positions(monkeypatch, kind, scalings):
    """A model's loss and gradients with tables for longer contexts against the oracle's, with the bounds that its unscaled tables have."""
    from olmax_amd import TransformerConfig
    sets = {"yarn": ops().RopeScaling("yarn", 4.0, original_length=32), "llama3": ops().RopeScaling("llama3", 8.0, original_length=64), "linear": ops().RopeScaling("linear", 2.0), None: None}
    per_layer, thetas = [sets[s] for s in scalings], [1e4, 5e5]
    qk = kind != "default"
    sizes = dict(n_heads=2, n_kv_heads=2, head_dim=64)
    ocfg = ref.ModelConfig(vocab=512, d_model=256, n_layers=2, hidden=512, layer_type="reordered" if qk else "pre", act="silu", qk_norm=qk, qk_norm_headwise=True, eps=1e-6, rope_theta_layers=thetas, **sizes)
    more = dict(rope_scaling=per_layer[0]) if scalings[0] == scalings[1] else dict(rope_scaling_per_layer=per_layer)
    hcfg = TransformerConfig(vocab_size=512, d_model=256, hidden_size=512, num_layers=2, layer_type=kind, qk_norm_headwise=qk, norm_eps=1e-6, rope_theta_per_layer=thetas, **sizes, **more)
    P = {k: (v + 0.1 * torch.randn(v.shape, generator=torch.Generator().manual_seed(3)) if "norm" in k else 2 * v).to(torch.bfloat16).double() for k, v in ref.init_params(ocfg, seed=1).items()}
    gen = torch.Generator().manual_seed(5)
    ids, labels = (torch.randint(0, 512, (2, 128), generator=gen, dtype=torch.int32) for _ in range(2))
    model = hcfg.build(batch_size=2, sequence_length=128)
    model.load_state_dict({k: v.float() for k, v in P.items()})
    loss = model.loss_and_grads(ids.cuda().reshape(-1), labels.cuda().reshape(-1)).item()
    monkeypatch.setattr(ref, "rope_tables", _scaled(dict(zip(thetas, per_layer))))
    rt = lambda t: t.to(torch.bfloat16).to(t.dtype)  # noqa: E731
    want, grads = ref.model_loss_and_grads(ocfg, P, ids, labels.long(), rt)
    assert abs(loss - want.item()) < 1e-2 * abs(want.item())
    for name, g in model.named_gradients().items():
        a, b = g.double().cpu().flatten(), grads[name].double().flatten()
        assert a @ b / (a.norm() * b.norm() + 1e-30) >= 0.999, name


@pytest.mark.parametrize("head_dim,dtype", [(1040, BF), (520, BF), (520, F32)])
def test_more_tokens_than_a_dimension_of_the_grid_has_threads_for(head_dim, dtype):
    """Heads so wide that a workgroup of 256 has one token (or three), and so many tokens that their workgroups have 2^32 threads and more: the first tokens, those about 2^23 and 2^24 workgroups, and
    the last against the plain form, in place; all others, which hold one number, against 37 rows of it."""
    per = 256 // (head_dim // (8 if dtype == BF else 4))
    T = per * 2 ** 24 + 5
    cos, sin = tables(60, 32)
    x = torch.full((T, head_dim), 3.0, dtype=dtype, device="cuda")
    at = torch.cat([torch.arange(max(0, m - 20), min(T, m + 20)) for m in (0, per * 2 ** 23, per * 2 ** 24)])
    some = torch.randn(at.numel(), head_dim, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[at.cuda()] = some.cuda()
    assert ops().rotary_fwd(x, cos, sin, heads=1, head_dim=head_dim, seq_len=37, out=x) is x
    check(x[at.cuda()], some, cos, sin, at % 37, 1, head_dim, "half", False)
    want = ops().rotary_fwd(torch.full((37, head_dim), 3.0, dtype=dtype, device="cuda"), cos, sin, heads=1, head_dim=head_dim)
    x[at.cuda()] = want[at.cuda() % 37]
    for first in range(0, T, 37 * 2 ** 15):  # all rows, each once
        chunk = x[first: first + 37 * 2 ** 15]
        n = chunk.shape[0] // 37 * 37
        assert (chunk[:n].view(-1, 37, head_dim) == want).all() and torch.equal(chunk[n:], want[: chunk.shape[0] - n]), first


def _model_of_scaled_positions(kind, per_layer, thetas=(1e4, 5e5)):
    qk = kind != "default"
    sizes = dict(n_heads=2, n_kv_heads=2, head_dim=64)
    ocfg = ref.ModelConfig(vocab=512, d_model=256, n_layers=2, hidden=512, layer_type="reordered" if qk else "pre", act="silu", qk_norm=qk, qk_norm_headwise=True, eps=1e-6,
                           rope_theta_layers=list(thetas), **sizes)
    gen = torch.Generator().manual_seed(5)
    ids, labels = (torch.randint(0, 512, (2, 128), generator=gen, dtype=torch.int32) for _ in range(2))
    P = {k: (v + 0.1 * torch.randn(v.shape, generator=torch.Generator().manual_seed(3)) if "norm" in k else 2 * v).to(BF).double() for k, v in ref.init_params(ocfg, seed=1).items()}
    more = dict(vocab_size=512, d_model=256, hidden_size=512, num_layers=2, layer_type=kind, qk_norm_headwise=qk, norm_eps=1e-6, rope_theta_per_layer=list(thetas),
                rope_scaling_per_layer=per_layer, **sizes)
    return ocfg, P, ids, labels, more


@pytest.mark.parametrize("kind", ["default", "reordered_norm"])
def test_a_models_gradients_are_as_large_as_the_tables_make_them(monkeypatch, kind):
    """Norms of a model's gradients with yarn's tables, whose size (1.139 here) enters the scores twice and the gradients of queries and keys again.  A cosine of 0.999 leaves an error of sqrt(0.002)
    across the gradient, and roundings leave no more along it: norms agree within 0.045.  The oracle with tables of size 1, and one that leaves the size out of the backward pass alone, do not."""
    from olmax_amd import TransformerConfig
    yarn = ops().RopeScaling("yarn", 4.0, original_length=32)
    ocfg, P, ids, labels, more = _model_of_scaled_positions(kind, [yarn, yarn])
    model = TransformerConfig(**more).build(batch_size=2, sequence_length=128)
    model.load_state_dict({k: v.float() for k, v in P.items()})
    model.loss_and_grads(ids.cuda().reshape(-1), labels.cuda().reshape(-1))
    got = {name: g.double().cpu().norm().item() for name, g in model.named_gradients().items()}
    rt = lambda t: t.to(BF).to(t.dtype)  # noqa: E731
    of = _scaled({1e4: yarn, 5e5: yarn})
    monkeypatch.setattr(ref, "rope_tables", of)
    want = {name: g.double().norm().item() for name, g in ref.model_loss_and_grads(ocfg, P, ids, labels.long(), rt)[1].items()}
    monkeypatch.setattr(ref, "rope_tables", lambda S, D, theta, dtype=F32: tuple((t.double() / yarn.size).to(dtype) for t in of(S, D, theta, torch.float64)))
    bare = {name: g.double().norm().item() for name, g in ref.model_loss_and_grads(ocfg, P, ids, labels.long(), rt)[1].items()}
    for name in want:
        assert abs(got[name] / want[name] - 1) < 0.045, (name, got[name], want[name])
    turned = [name for name in want if "q_proj" in name or "k_proj" in name or "q_norm" in name or "k_norm" in name]
    assert len(turned) == (4 if kind == "default" else 8)
    for name in turned:  # planted in the oracle: the forward's size, and the backward's
        assert abs(bare[name] / want[name] - 1) > 0.045 and abs(1 / yarn.size - 1) > 2 * 0.045, (name, bare[name], want[name])


def test_a_layer_has_its_own_scaling():
    """One layer by itself takes the tables that the model gives it."""
    from olmax_amd import TransformerConfig
    from olmax_amd.layer import TransformerBlock
    yarn = ops().RopeScaling("yarn", 4.0, original_length=32)
    *_, more = _model_of_scaled_positions("default", [None, yarn])
    c = TransformerConfig(**more)
    for i, want in enumerate((ops().rope_tables(128, 64, 1e4, "cuda"), ops().rotary_tables(128, 64, 5e5, "cuda", scaling=yarn))):
        block = TransformerBlock(c, layer_idx=i, batch_size=2, sequence_length=128)
        assert torch.equal(block.cos, want[0]) and torch.equal(block.sin, want[1])
