"""More of what the entry points of log probabilities and distillation refuse.  No GPU needed: addresses are never read."""
import pytest

from test_logprobs import ARG, CALLS, _lib


@pytest.mark.parametrize("softcap", [1e-45, 1e-39, 9e-31, 1.1e30, float("inf")])
@pytest.mark.parametrize("name", CALLS)
def test_softcaps_whose_factor_fp32_has_not(name, softcap):
    lib = _lib()
    assert lib.typed(name)(*{**CALLS[name], "softcap": softcap}.values()) == ARG
    assert b"softcap" in lib.load().olmax_last_error_string()


# pointers that may not be null, besides those of the calls' own list (an optional one of another call has the same name)
NEEDED = [("olmax_token_logprobs_bwd", "dlogits"), ("olmax_token_logprobs", "logprobs_targets"), ("olmax_token_logprobs", "top_ids"), ("olmax_token_logprobs", "top_logprobs"),
          ("olmax_lmhead_logprobs", "workspace"), ("olmax_lmhead_logprobs_bwd", "workspace"), ("olmax_lmhead_distill", "workspace"), ("olmax_distill", "workspace"),
          ("olmax_lmhead_logprobs_bwd", "dh_dW")]
GROUPS = {"logprobs_targets": ("targets",), "dh_dW": ("dh", "dW")}  # log probabilities without targets; neither gradient


@pytest.mark.parametrize("name,what", NEEDED)
def test_null_pointers(name, what):
    lib = _lib()
    null = GROUPS.get(what, (what,))
    assert all(n in CALLS[name] for n in null)
    rc = lib.typed(name)(*{**CALLS[name], **dict.fromkeys(null)}.values())
    assert rc == ARG, lib.load().olmax_last_error_string()
    assert name.encode() in lib.load().olmax_last_error_string()
