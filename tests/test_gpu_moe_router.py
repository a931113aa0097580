"""The types a mixture's router may have."""
import pytest
import torch
import torch.nn.functional as F

from sparseflow_b200.nn import SparseFlowMoE

from .operator_refs import gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("router", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
def test_router_types(router):
    g, E, H, I, dt = gen(1), 6, 128, 64, torch.bfloat16
    wr, bias = randn(g, E, H, scale=0.3).to(router), randn(g, E).to(router)
    m = SparseFlowMoE(wr, randn(g, E, I, H, dtype=dt, scale=0.06), randn(g, E, I, H, dtype=dt, scale=0.06), randn(g, E, H, I, dtype=dt, scale=0.06), 2,
                      router_bias=bias)
    x = randn(g, 33, H, dtype=dt)
    logits = F.linear(x.to(router), wr, bias).float()
    assert torch.equal(m.route(x).experts.long(), logits.sort(dim=1, descending=True, stable=True).indices[:, :2])
    assert m(x).shape == (33, H) and m(x).isfinite().all()
