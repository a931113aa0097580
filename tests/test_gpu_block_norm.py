"""Norms between two blocks, fused with gate, scale and sum, against a 64-bit reference."""
import pytest
import torch

from sparseflow_b200 import ops
from sparseflow_b200.nn import SparseFlowBlockNorm

from .operator_refs import DT, block_norm_ref, close, gen, randn

pytestmark = pytest.mark.gpu


def _run(x, y, kind="rms", weight=None, bias=None, post_weight=None, post_bias=None, gate=None, scale=0.75, eps=1e-5, post_eps=1e-3):
    r, h = ops.block_norm(x, y, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate, scale=scale, eps=eps, post_eps=post_eps, kind=kind)
    rr, rs, hr, hs = block_norm_ref(x, y, weight, bias, post_weight, post_bias, gate, scale, eps, post_eps, kind)
    close(r, rr, rs)
    if weight is None:
        assert h is None
    else:
        close(h, hr, hs)
    return r, h


WIDTHS = [1, 7, 8, 64, 65, 250, 256, 257, 511, 520, 1000, 1001, 2048, 4096, 4097, 8191, 8192, 12345, 16376, 16383, 16384]


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dt,stream", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
def test_widths(H, kind, dt, stream):
    g = gen(H)
    t = DT[dt]
    x, y = randn(g, 11, H, dtype=DT[stream], scale=3.0), randn(g, 11, H, dtype=t)
    v = [randn(g, H, dtype=t) for _ in range(5)]
    layer = kind == "layer"
    _run(x, y, kind, weight=v[0], bias=v[1] if layer else None, post_weight=v[2], post_bias=v[3] if layer else None, gate=v[4])
    _run(x, y, kind, weight=v[0])
    _run(x, None, kind, weight=v[0], bias=v[1])


@pytest.mark.parametrize("rows,gates", [(1, 1), (12, 4), (12, 12), (300, 3)])
@pytest.mark.parametrize("H", [200, 1001, 2056])
@pytest.mark.parametrize("post", [False, True])
def test_gates_and_rows(rows, gates, H, post):
    g = gen(rows + H)
    x, y, w = randn(g, rows, H, dtype=torch.bfloat16), randn(g, rows, H, dtype=torch.bfloat16), randn(g, H, dtype=torch.bfloat16)
    pw = randn(g, H, dtype=torch.bfloat16) if post else None
    for gate in (randn(g, gates, H, dtype=torch.bfloat16), randn(g, gates, 1, dtype=torch.bfloat16), randn(g, gates, H + 8, dtype=torch.bfloat16)[:, 8:], None):
        _run(x, y, weight=w, post_weight=pw, gate=gate)
    _run(x, y, weight=None, post_weight=pw, post_bias=pw)      # no second norm


@pytest.mark.parametrize("H", [2056, 2057, 4096, 4099, 8192, 8185, 12345, 16368, 16370])
@pytest.mark.parametrize("kind,dt,stream", [("rms", "bf16", "f32"), ("layer", "f16", "f16"), ("rms", "f32", "f32")])
def test_more_rows_than_blocks(H, kind, dt, stream):
    """Blocks that stay and fetch their next row while they reduce one; the last row ends inside a piece."""
    g = gen(H)
    t, n = DT[dt], 1503
    x, y = randn(g, n, H, dtype=DT[stream]), randn(g, n, H, dtype=t)
    v = [randn(g, H, dtype=t) for _ in range(4)]
    _run(x, y, kind, weight=v[0], bias=v[1], post_weight=v[2], post_bias=v[3], gate=v[1])
    _run(x, y, kind, weight=v[0], gate=randn(g, 3, H, dtype=t))
    _run(x, y, kind, post_weight=v[2])
    _run(x, y, kind)
    _run(x, None, kind, weight=v[0])


@pytest.mark.parametrize("H,pitch,at", [(64, 80, 0), (64, 80, 3), (1001, 1009, 0), (1001, 1001, 0), (1000, 1003, 1), (4097, 4105, 0)])
def test_strides(H, pitch, at):
    g = gen(H + pitch)
    make = lambda p: randn(g, 9, p + 8, dtype=torch.float16)[:, at:at + H]  # noqa: E731
    w = randn(g, H + 1, dtype=torch.float16)
    _run(make(pitch), make(pitch), weight=w[:H])
    _run(make(pitch), make(pitch + 8), weight=w[1:], gate=w[:H])      # rows that lie otherwise, unaligned weights
    _run(randn(g, H, 9, dtype=torch.float16).t(), make(pitch), weight=w[:H])
    _run(make(pitch)[:1].expand(9, H), make(pitch), weight=w[:H])     # one row for all


def test_values():
    H = 4096
    g = gen(3)
    w = randn(g, H)
    _run(1000 + randn(g, 4, H), randn(g, 4, H), "layer", weight=w)    # a large mean costs no digits
    _run(torch.zeros(3, H, device="cuda"), torch.zeros(3, H, device="cuda"), weight=w, post_weight=w)
    x = randn(g, 3, H, dtype=torch.bfloat16)
    x[1, 5] = torch.nan
    x[2, 7] = torch.inf
    r, h = ops.block_norm(x, torch.zeros_like(x), weight=w.bfloat16())
    assert torch.isfinite(h[0]).all() and torch.isnan(h[1]).all() and torch.isnan(h[2, 7]) and (h[2, :7] == 0).all()
    assert torch.equal(torch.isnan(r), torch.isnan(x))


def test_module_and_empty():
    g = gen(4)
    x, y, w = randn(g, 2, 5, 96, dtype=torch.bfloat16), randn(g, 2, 5, 96, dtype=torch.bfloat16), randn(g, 96, dtype=torch.bfloat16)
    m = SparseFlowBlockNorm(w, post_weight=w, gate=w, scale=0.5)
    r, h = m(x, y)
    r2, h2 = ops.block_norm(x.view(10, 96), y.view(10, 96), weight=w, post_weight=w, gate=w, scale=0.5)
    assert r.shape == x.shape and torch.equal(r.view(10, 96), r2) and torch.equal(h.view(10, 96), h2)
    r, h = m(x)
    assert torch.equal(r, x) and torch.equal(h.view(10, 96), ops.block_norm(x.view(10, 96), weight=w)[1])
    per_sequence = randn(g, 2, 96, dtype=torch.bfloat16)
    assert torch.equal(m(x, y, gate=per_sequence)[0][1], m(x[1:], y[1:], gate=per_sequence[1:])[0][0])
    r, h = ops.block_norm(x.view(10, 96)[:0], y.view(10, 96)[:0], weight=w)
    assert r.shape == h.shape == (0, 96)


def test_refusals():
    g = gen(5)
    x, w = randn(g, 4, 64, dtype=torch.bfloat16), randn(g, 64, dtype=torch.bfloat16)
    bad = [
        lambda: ops.block_norm(x.cpu(), weight=w), lambda: ops.block_norm(x, weight=None), lambda: ops.block_norm(x, x, weight=w, kind="batch"),
        lambda: ops.block_norm(x.double(), weight=w), lambda: ops.block_norm(x, x.half(), weight=w.half()), lambda: ops.block_norm(x, x[:3], weight=w),
        lambda: ops.block_norm(x, x, weight=w[:63]), lambda: ops.block_norm(x, x, weight=w.float()), lambda: ops.block_norm(x, x, weight=w.cpu()),
        lambda: ops.block_norm(x, weight=w, gate=w), lambda: ops.block_norm(x, weight=w, post_weight=w), lambda: ops.block_norm(x, x, weight=None, bias=w),
        lambda: ops.block_norm(x, x, weight=w, post_bias=w), lambda: ops.block_norm(x, x, weight=w, gate=x[:3]), lambda: ops.block_norm(x, x, weight=w, gate=x[:, :2]),
        lambda: ops.block_norm(randn(g, 1, 16385, dtype=torch.bfloat16), weight=randn(g, 16385, dtype=torch.bfloat16)), lambda: ops.block_norm(w, weight=w),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
