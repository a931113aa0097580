"""Weights of more than a million rows: 256 experts of a few thousand, compressed in one launch."""
import pytest
import torch

from sparseflow_b200 import ops, serialize

from .operator_refs import close, gen, randn

pytestmark = pytest.mark.gpu

E, K = 256, 64


def _same(got, want):
    assert torch.equal(got.values.view(torch.int16), want.values.view(torch.int16)) and torch.equal(got.meta, want.meta)


@pytest.mark.parametrize("N", [4096, 4224])      # 65536 groups of 16 rows, and more
def test_experts(N):
    g = gen(N)
    w = randn(g, E, N, K, dtype=torch.bfloat16)
    cw = ops.compress_experts(w)
    for e in (0, 1, 100, 248, 254, 255):
        _same(cw.expert(e), ops.compress_weight(w[e]))
    sizes = torch.randint(0, 3, (E,), generator=g, device="cuda")
    sizes[-1] = 3
    groups = ops.group_rows(torch.repeat_interleave(torch.arange(E, device="cuda"), sizes), E)
    x = randn(g, groups.rows.numel(), K, dtype=torch.bfloat16)
    y = ops.grouped_sparse_gemm(x, cw, groups)
    assert ops.device_status() == 0
    off = groups.offsets.tolist()
    for e in (0, 128, 254, 255):
        pruned = ops.prune_compress_24(w[e], want_values=False, want_meta=False, want_pruned=True)["pruned"].double()
        xe = x[off[e]:off[e + 1]].double()
        close(y[off[e]:off[e + 1]], xe @ pruned.t(), xe.abs() @ pruned.abs().t() * K * 2.0 ** -24)      # a rounding per term


def test_gate_up_experts():
    g = gen(2)
    gate, up = randn(g, E, 2112, K, dtype=torch.float16), randn(g, E, 2112, K, dtype=torch.float16)
    cw = ops.compress_gate_up_experts(gate, up)
    for e in (0, 7, 247, 248, 255):
        _same(cw.expert(e), ops.compress_gate_up(gate[e], up[e]))


def test_one_weight():
    w = randn(gen(3), 1_100_000, K, dtype=torch.float16)
    whole = ops.prune_compress_24(w, want_ref_codes=True, want_pruned=True)
    part = ops.prune_compress_24(w[-1_100_000 % 128 - 4096:], want_ref_codes=True, want_pruned=True)      # the last tiles
    for name, n in (("values", K // 2), ("ref_codes", K // 4), ("pruned", K)):
        a, b = whole[name].reshape(-1, n), part[name].reshape(-1, n)
        assert torch.equal(a[-4000:], b[-4000:])
    m = part["meta"].numel()
    assert torch.equal(whole["meta"][-m:], part["meta"])
    blob, valid = serialize.compress_checked(whole["pruned"])
    assert valid
    back = serialize.unpack(blob)
    assert torch.equal(back.values, whole["values"]) and torch.equal(back.meta, whole["meta"])
