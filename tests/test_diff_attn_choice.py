"""Which forms differential attention takes (no GPU needed), and that the GPU tests reach each of them."""
import pytest

import test_diff_attn_forms_gpu as large
import test_diff_attn_gpu as small


def form(B, S, H, KH, D, window=None):
    from olmax_amd import _lib
    if not _lib.lib_path().exists():
        pytest.skip("libolmax_hip.so not built")
    return _lib.load().olmax_diff_attn_form(B, S, H, KH, D, -1 if window is None else window)


@pytest.mark.parametrize("call", large.FORMS)
def test_large_calls_take_the_forms_that_they_are_tests_of(call):
    assert form(*call[:6]) == call[6]


def test_every_form_is_reached():
    """For heads of 32 and 64: each form of the forward pass, each of dQ with chains short and long (dealt out ones are long), each of dK/dV, and each with and without a window and with several query
    heads to a key head."""
    calls = [c[:6] for c in large.FORMS] + [s[:6] for s in small.SHAPES]
    for D in (32, 64):
        at = [(form(*c), c) for c in calls if c[4] == D]
        fwd, dq = {f & 3 for f, _ in at}, {f >> 2 & 7 for f, _ in at}
        assert fwd == ({1, 2} if D == 32 else {0, 1, 2}) and dq == {0, 1, 4, 5, 6}
        kinds = {0, 1, 2, 4} if D == 32 else {0, 1, 4}
        assert {f >> 5 for f, _ in at} == kinds
        assert {f >> 5 for f, c in at if c[2] > c[3]} == kinds
        assert {(f >> 2 & 5, f >> 5) for f, c in at if c[5] is not None} >= {(4, 0), (4, 1)}


def test_refused_shapes_have_no_form():
    assert form(1, 10, 4, 4, 128) == form(1, 10, 3, 2, 64) == form(0, 10, 4, 4, 64) == form(1, 0, 4, 4, 64) == -1
    for window in (1100, 2 ** 31 - 1):  # past the first key: none
        assert form(1, 1100, 4, 4, 64, window) == form(1, 1100, 4, 4, 64)
