"""The plain form of distillation where the teacher's tokens lead by so much that the probability of all others together leaves the range of its type.  No GPU needed."""
import math

import pytest
import torch

from oracle import ref


def test_half_a_probability_for_the_others():
    """One token with q = 1/2 against 999 equal ones 80 nats behind: p is 1 and 0, the loss ln(1/2) + lead / 2 - ln(999) / 2, each other token's gradient -1/2 of 1/999."""
    z = torch.zeros(1, 1000, dtype=torch.float64)
    z[0, 7] = 80.0
    ids, t = torch.tensor([[7]]), torch.tensor([[math.log(0.5)]], dtype=torch.float64)
    loss, d = (f(z, ids, t, tail="bucket", reduction="none")[0] for f in (ref.distill_fwd, ref.distill_bwd))
    assert abs(loss - (math.log(0.5) + 40.0 - math.log(999) / 2)) < 1e-12
    assert abs(d[7] - 0.5) < 1e-12 and (d[8:] + 0.5 / 999).abs().max() < 1e-15


@pytest.mark.parametrize("lead", [0.0, 60.0, 85.0, 120.0, 800.0, 8192.0])
@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (0.05, 0.0), (1e-3, 2.0)])
def test_the_others_gradient_is_autograds(lead, temperature, softcap):
    """64 bits through some 20 operations on scores of up to `size`, whose differences lose 2^-53 of it: 1e-13 (1 + size)."""
    z = torch.randn(4, 40, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    ids = torch.tensor([[3, 9, 20], [0, 39, 1], [5, 5, 6], [-1, 2, 3]])
    t = torch.tensor([[0.5, 0.2, 0.1], [0.3, 0.3, 0.3], [0.9, 0.5, 0.05], [0.1, 0.1, 0.1]], dtype=torch.float64).log()
    for row in range(3):
        z[row, ids[row]] += lead
    z.requires_grad_()
    kw = dict(tail="bucket", temperature=temperature, softcap=softcap, reduction="none")
    dl = torch.tensor([1.0, -2.0, 0.5, 3.0], dtype=torch.float64)
    (ref.distill_fwd(z, ids, t, **kw) * dl).sum().backward()
    got = ref.distill_bwd(z.detach(), ids, t, dloss=dl, **kw)
    size = (softcap if softcap else 8.0 + lead) / temperature
    assert torch.isfinite(got).all() and (got - z.grad).abs().max() < 1e-13 * (1 + size) / temperature


def test_no_other_token_is_left():
    """Nothing pulls on tokens of minus infinity; the loss says what it costs to rule them out."""
    z = torch.full((2, 9), -math.inf, dtype=torch.float64)
    z[:, 4] = 1.0
    z[1, 5] = 1.0
    ids, t = torch.tensor([[4], [4]]), torch.full((2, 1), math.log(0.75), dtype=torch.float64)
    loss, d = (f(z, ids, t, tail="bucket", reduction="none") for f in (ref.distill_fwd, ref.distill_bwd))
    assert loss[0] == math.inf and torch.isfinite(loss[1]) and torch.isfinite(d).all()
    assert (d[0, :4] == 0).all() and abs(d[1].sum()) < 1e-15 and abs(d[1, 5] - (0.5 - 0.25)) < 1e-15


def test_others_at_the_types_lowest_value():
    """A mask of finite numbers leads as any other: each of the others has its equal share of r."""
    z = torch.full((1, 50), float(torch.finfo(torch.float32).min), dtype=torch.float64)
    z[0, 3] = 1.0
    d = ref.distill_bwd(z, torch.tensor([[3]]), torch.full((1, 1), math.log(0.75), dtype=torch.float64), tail="bucket", temperature=0.5, reduction="none")[0]
    assert abs(d[3] - 0.5) < 1e-15 and (d[4:] + 0.5 / 49).abs().max() < 1e-15
