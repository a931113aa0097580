"""The prefill command at sizes and with checks that its arms need."""
import pytest

from sparseflow_b200 import ops, prefill_e2e

pytestmark = pytest.mark.gpu


def test_hidden_sizes_beyond_the_fused_norms():
    """The arm with fused norms is left out; the others run as they did before there was one."""
    hidden = ops.MAX_NORM_COLS + 64
    r = prefill_e2e.run(layers=1, hidden=hidden, inter=64, heads=hidden // 64, batch=1, seq=16, iters=1, warmup=1)
    assert r["mlp_layers_replaced"] == 1 and "sparse_mlp_attn" in r["arms"] and "fused_norms" not in r["arms"]
