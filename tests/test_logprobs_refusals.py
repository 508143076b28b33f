"""More of what the entry points of log probabilities and distillation refuse.  No GPU needed: addresses are never read."""
import pytest

from test_logprobs import ARG, CALLS, _lib


@pytest.mark.parametrize("softcap", [1e-45, 1e-39, 9e-31, 1.1e30, float("inf")])
@pytest.mark.parametrize("name", CALLS)
def test_softcaps_whose_factor_fp32_has_not(name, softcap):
    lib = _lib()
    assert lib.typed(name)(*{**CALLS[name], "softcap": softcap}.values()) == ARG
    assert b"softcap" in lib.load().olmax_last_error_string()
