"""Logits that compare equal are a tie, which goes to the lowest expert, whatever their sign bits."""
import pytest
import torch

from sparseflow_b200 import ops

from .operator_refs import DT, gen, group_ref, route_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,E,k", [(1, 2, 1), (7, 5, 3), (40, 64, 8), (300, 128, 6), (33, 1000, 32)])
@pytest.mark.parametrize("renorm", [True, False])
def test_signed_zeros(dt, n, E, k, renorm):
    """Rows of +0 and -0 in any order, with a few numbers on either side: the choice cuts through the tie."""
    g = gen(n + E + k)
    sign = torch.where(torch.rand(n, E, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    logits = sign * 0.0
    if E > 4:      # one above the zeros, some below
        logits[:, E // 2] = 1.5
        logits[:, 1] = -2.0
    logits[0, 0], logits[0, 1] = -0.0, 0.0
    logits = logits.to(DT[dt])
    r = ops.moe_route(logits, k, renormalize=renorm)
    weights, experts = route_ref(logits, k, renorm)
    assert torch.equal(r.experts.cpu(), experts)
    # exp of 0, of 1.5 and of 2 from the largest, sums of at most 1000 terms in 32 + 5 levels, one division
    assert ((r.weights.cpu().double() - weights).abs() <= 64 * 2.0 ** -24 * weights).all()
    for got, want in zip((r.groups.offsets, r.groups.rows, r.groups.slots), group_ref(experts, E, k)):
        assert torch.equal(got.cpu(), want)
