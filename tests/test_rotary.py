"""Rotary positions: what the entry points and their wrappers refuse.  No GPU needed: addresses are never read."""
import math

import pytest

ARG, SHAPE, ALIGN = -1, -2, -3
AT = 1 << 20  # an address


def lib():
    from olmax_amd import _lib
    if not _lib.lib_path().exists():
        pytest.skip("libolmax_hip.so not built")
    return _lib


GOOD = dict(stream=None, x=AT, y=AT * 9, cos=AT * 20, sin=AT * 30, positions=None, tokens=8, heads=4, head_dim=64, rotary_dim=64, table_rows=16, seq_len=16, ldx=256, ldy=256, layout=0,
            f32=0)
REFUSED = [
    (dict(x=None), ARG, b"null"), (dict(y=None), ARG, b"null"), (dict(cos=None), ARG, b"null"), (dict(sin=None), ARG, b"null"),
    (dict(tokens=-1), SHAPE, b"shape"), (dict(tokens=1 << 31), SHAPE, b"shape"), (dict(heads=0), SHAPE, b"shape"), (dict(head_dim=0), SHAPE, b"shape"),
    (dict(heads=1 << 20, head_dim=64), SHAPE, b"shape"), (dict(rotary_dim=0), SHAPE, b"rotary_dim"), (dict(rotary_dim=-2), SHAPE, b"rotary_dim"),
    (dict(rotary_dim=63), SHAPE, b"rotary_dim"), (dict(rotary_dim=66), SHAPE, b"rotary_dim"), (dict(table_rows=0), SHAPE, b"seq_len"), (dict(seq_len=0), SHAPE, b"seq_len"),
    (dict(seq_len=17), SHAPE, b"seq_len"), (dict(seq_len=-1), SHAPE, b"seq_len"), (dict(ldx=255), SHAPE, b"overlap"), (dict(ldy=-256), SHAPE, b"overlap"),
    (dict(ldx=1 << 31), SHAPE, b"2^31"), (dict(layout=2), ARG, b"layout"), (dict(layout=-1), ARG, b"layout"), (dict(x=AT + 1), ALIGN, b"aligned"), (dict(y=AT * 9 + 1), ALIGN, b"aligned"),
    (dict(x=AT + 2, f32=1), ALIGN, b"aligned"), (dict(cos=AT + 2), ALIGN, b"aligned"), (dict(sin=AT + 1), ALIGN, b"aligned"), (dict(positions=AT + 2), ALIGN, b"aligned"),
    (dict(y=AT, ldy=264), ARG, b"in place"), (dict(y=AT + 2), ARG, b"overlaps"), (dict(y=AT + 256), ARG, b"overlaps"), (dict(y=AT - 512), ARG, b"overlaps"),
    (dict(y=AT + 512, ldx=512, ldy=768), ARG, b"overlaps"),
]


@pytest.mark.parametrize("name", ["olmax_rotary_fwd", "olmax_rotary_bwd"])
@pytest.mark.parametrize("change,code,word", REFUSED)
def test_rotation_refuses(name, change, code, word):
    L = lib()
    assert L.typed(name)(*{**GOOD, **change}.values()) == code
    said = L.load().olmax_last_error_string()
    assert word in said and name.encode() in said


def test_no_tokens_are_no_work():
    L = lib()
    assert L.typed("olmax_rotary_fwd")(*{**GOOD, "tokens": 0, "x": None, "y": None}.values()) == 0


TABLES = dict(cos=AT, sin=AT * 2, length=16, rotary_dim=64, theta=1e4, kind=0, factor=1.0, original=8192.0, low=1.0, high=4.0, size=1.0)
TABLES_REFUSED = [
    (dict(cos=0), ARG), (dict(sin=0), ARG), (dict(length=0), SHAPE), (dict(length=1 << 31), SHAPE), (dict(rotary_dim=0), SHAPE), (dict(rotary_dim=3), SHAPE), (dict(rotary_dim=514), SHAPE),
    (dict(theta=1.0), ARG), (dict(theta=-5.0), ARG), (dict(theta=math.nan), ARG), (dict(theta=math.inf), ARG), (dict(kind=-1), ARG), (dict(kind=4), ARG), (dict(kind=1, factor=0.5), ARG),
    (dict(kind=1, factor=math.nan), ARG), (dict(kind=2, factor=2e6), ARG), (dict(kind=2, original=0.0), ARG), (dict(kind=3, original=math.nan), ARG), (dict(kind=2, low=0.0), ARG),
    (dict(kind=2, low=4.0), ARG), (dict(kind=3, low=math.nan), ARG), (dict(kind=3, high=0.5), ARG), (dict(kind=2, high=math.inf), ARG), (dict(size=0.0), ARG), (dict(size=math.nan), ARG),
]


@pytest.mark.parametrize("change,code", TABLES_REFUSED)
def test_tables_refuse(change, code):
    L = lib()
    a = {**TABLES, **change}
    assert L.typed("olmax_rotary_tables")(None, *a.values()) == code and b"olmax_rotary_tables" in L.load().olmax_last_error_string()


def test_argument_types_of_the_tables_match_the_header():
    import re
    from pathlib import Path
    _lib = lib()
    text = re.sub(r"/\*.*?\*/", "", (Path(__file__).resolve().parent.parent / "include" / "olmax_hip.h").read_text(), flags=re.S)
    for name, letters in _lib._SIGNATURES_OF_64_BITS.items():
        args = re.search(name + r"\s*\(([^;]*)\)\s*;", text)[1]
        kinds = ["P" if "*" in a or "olmax_stream_t" in a else {"int32_t": "I", "int64_t": "L", "float": "F", "double": "D"}[a.split()[0]] for a in args.split(",")]
        assert "".join(kinds) == letters, name


def test_scalings_by_name():
    from olmax_amd.ops import RopeScaling
    assert RopeScaling("linear", 2.0).c_args()[:2] == (1, 2.0)
    assert RopeScaling("llama3", 8.0, original_length=4096).c_args() == (2, 8.0, 4096, 1.0, 4.0, 1.0)
    kind, factor, length, low, high, size = RopeScaling("yarn", 4.0).c_args()
    assert (kind, factor, length, low, high) == (3, 4.0, 8192, 1.0, 32.0) and size == pytest.approx(0.1 * math.log(4.0) + 1.0)
    assert RopeScaling("yarn", 4.0, attention_factor=1.25).c_args()[5] == 1.25
    with pytest.raises(ValueError):
        RopeScaling("dynamic", 2.0)
    with pytest.raises(ValueError):
        RopeScaling("linear", 2.0, attention_factor=1.0)


def test_wrappers_refuse_cpu_tensors():
    import torch

    from olmax_amd import ops
    from olmax_amd._lib import OlmaxHipError
    x, t = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(4, 32)
    for call in (ops.rotary_fwd, ops.rotary_bwd):
        with pytest.raises(OlmaxHipError):
            call(x, t, t, heads=1, head_dim=64)
    with pytest.raises(OlmaxHipError):
        ops.rotary_tables(4, 64, 1e4, "cpu")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_plain_rotation_and_its_gradient(layout):
    """A turn keeps lengths and the angle between two rows of one distance; its gradient is autograd's.  float64, a handful of operations: 1e-13."""
    import torch

    from oracle import ref
    g = torch.Generator().manual_seed(0)
    angle = torch.arange(50, dtype=torch.float64)[:, None] * ref.rotary_freqs(8, 1e4)
    c, s = angle.cos(), angle.sin()
    x = torch.randn(4, 2 * 12, generator=g, dtype=torch.float64, requires_grad=True)
    kw = dict(heads=2, head_dim=12, layout=layout)
    p = torch.tensor([3, 20, -1, 0])
    y = ref.rotary(x, c, s, p, **kw)
    dy = torch.randn(4, 24, generator=g, dtype=torch.float64)
    assert (torch.autograd.grad(y, x, dy)[0] - ref.rotary(dy, c, s, p, back=True, **kw)).abs().max() < 1e-13
    x, y = x.detach().view(4, 2, 12), y.detach().view(4, 2, 12)
    assert torch.equal(y[2:], x[2:]) and torch.equal(y[..., 8:], x[..., 8:]) and (y.norm(dim=-1) - x.norm(dim=-1)).abs().max() < 1e-13
    moved = ref.rotary(x.reshape(4, 24), c, s, p + 17, **kw).view(4, 2, 12)
    assert ((moved[0] * moved[1]).sum() - (y[0] * y[1]).sum()).abs() < 1e-12
    a, b = (slice(0, 4), slice(4, 8)) if layout == "half" else (slice(0, 8, 2), slice(1, 8, 2))
    z = torch.complex(x[..., a], x[..., b])[:2] * torch.polar(torch.ones(()).double(), angle[p[:2]])[:, None]
    assert (y[:2, :, a] - z.real).abs().max() < 1e-13 and (y[:2, :, b] - z.imag).abs().max() < 1e-13


def test_plain_frequencies():
    import torch

    from oracle import ref
    f = ref.rotary_freqs(64, 5e5)
    assert f[0] == 1 and f[16] == pytest.approx(5e5 ** -0.5)
    assert torch.equal(ref.rotary_freqs(64, 5e5, kind="linear", factor=4.0) * 4, f)
    s = ref.rotary_freqs(64, 5e5, kind="llama3", factor=8.0)
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(s[turns >= 4], f[turns >= 4]) and torch.equal(s[turns <= 1], f[turns <= 1] / 8) and ((s < f) & (s > f / 8))[(turns > 1) & (turns < 4)].all()
    y = ref.rotary_freqs(64, 1e4, kind="yarn", factor=4.0, original_length=4096, high_turns=32.0)
    f = ref.rotary_freqs(64, 1e4)
    assert y[0] == f[0] and y[-1] == f[-1] / 4 and (y[1:] < y[:-1]).all()
