"""The prefill command at sizes and with checks that its arms need."""
import math

import pytest

from sparseflow_b200 import ops, prefill_e2e

pytestmark = pytest.mark.gpu


def test_hidden_sizes_beyond_the_fused_norms():
    """The arm with fused norms is left out; the others run as they did before there was one."""
    hidden = ops.MAX_NORM_COLS + 64
    r = prefill_e2e.run(layers=1, hidden=hidden, inter=64, heads=hidden // 64, batch=1, seq=16, iters=1, warmup=1)
    assert r["mlp_layers_replaced"] == 1 and "sparse_mlp_attn" in r["arms"] and "fused_norms" not in r["arms"]


@pytest.mark.parametrize("experts,top_k", [(0, 2), (4, 2), (8, 3)])
def test_errors_of_the_arms(experts, top_k):
    """With experts a rounding may send a token elsewhere, and the largest error is that token's; the median over the tokens is not.

    Two layers of MLP, each off by 8 half steps of the largest value (gate, up, their product, hidden values, an expert's row and the
    result on either side), two sums and the last norm with a half step on either side: 20 half steps of 2^-8.  Fused norms: five
    norms, each read with three roundings more or less."""
    r = prefill_e2e.run(layers=2, hidden=256, inter=512, heads=4, batch=1, seq=64, iters=1, warmup=1, experts=experts, top_k=top_k)
    assert math.isfinite(r["sparse_vs_pruned_dense_max_err_over_max"]) and math.isfinite(r["fused_norms_max_err_over_max"])
    assert r["sparse_vs_pruned_dense_median_token_err_over_max"] <= 20 * 2.0 ** -8
    assert r["fused_norms_median_token_err_over_max"] <= 15 * 2.0 ** -8
