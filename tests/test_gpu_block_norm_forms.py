"""The form of a block norm follows the rows per SM of the device: both sides of each border against the 64-bit form."""
import pytest
import torch

from sparseflow_b200 import ops

from .operator_refs import block_norm_ref, close, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [4096, 4099, 12352])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("per_sm", [1, 4])      # a piece per thread; blocks that stay
def test_borders(H, kind, per_sm):
    border = per_sm * torch.cuda.get_device_properties(0).multi_processor_count
    g = gen(H + per_sm)
    x, y, w = randn(g, border + 1, H), randn(g, border + 1, H, dtype=torch.bfloat16), randn(g, H, dtype=torch.bfloat16)
    for n in (border - 1, border, border + 1):
        r, h = ops.block_norm(x[:n], y[:n], weight=w, post_weight=w, kind=kind)
        rr, rs, hr, hs = block_norm_ref(x[:n], y[:n], w, None, w, None, None, 1.0, 1e-5, 1e-5, kind)
        close(r, rr, rs)
        close(h, hr, hs)
