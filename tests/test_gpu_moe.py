"""Router, grouping, grouped sparse products and the weighted sum of the experts' rows against 64-bit references."""
import pytest
import torch

from sparseflow_b200 import _lib, ops

from .operator_refs import DT, close, gen, group_ref, randn, route_ref

pytestmark = pytest.mark.gpu


def _same(groups, ref):
    for got, want in zip((groups.offsets, groups.rows, groups.slots), ref):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("n,groups,per_row", [(0, 3, 1), (1, 1, 1), (31, 7, 1), (512, 64, 4), (513, 1024, 1), (4096, 5, 8), (4098, 3, 6), (20001, 128, 1)])
def test_group_rows(n, groups, per_row):
    ids = torch.randint(-2, groups + 2, (n,), generator=gen(n + groups), device="cuda")      # some of no group
    if n > 10:
        ids[3:9] = 0                                                                          # and one group several times over
    _same(ops.group_rows(ids.to(torch.int32), groups, per_row), group_ref(ids, groups, per_row))
    _same(ops.group_rows(ids * 1, groups, per_row), group_ref(ids, groups, per_row))          # int64


def test_group_rows_none_and_far_ids():
    ids = torch.tensor([-1, 2 ** 40, -2 ** 40, 2 ** 32, 7], device="cuda")                    # 2**32 would wrap to group 0
    _same(ops.group_rows(ids, 4), group_ref(torch.tensor([-1] * 5), 4))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,E,k", [(0, 4, 2), (1, 1, 1), (5, 3, 3), (32, 64, 6), (33, 32, 4), (70, 33, 5), (300, 128, 8), (130, 200, 8), (40, 1000, 32), (700, 8, 2)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route(dt, n, E, k, renorm):
    g = gen(n + E + k)
    logits = randn(g, n, E, dtype=DT[dt], scale=2.0)           # 16-bit logits: many ties
    if n > 4:
        logits[1] = -torch.inf                                  # padding: goes nowhere
        logits[2, : E - 1] = -torch.inf                         # fewer experts than asked for
        logits[3] = 0.5                                         # all equal
        logits[4, ::2] = torch.nan
    wide = torch.zeros(n, E + 3, dtype=DT[dt], device="cuda")   # rows of a wider tensor
    wide[:, 1:E + 1] = logits
    r = ops.moe_route(wide[:, 1:E + 1], k, renormalize=renorm)
    weights, experts = route_ref(logits, k, renorm)
    assert torch.equal(r.experts.cpu(), experts)
    # exp: two steps, its argument |difference| <= 20 roundings, the sum of up to 1024 in 32 + 5 levels, one division
    assert ((r.weights.cpu().double() - weights).abs() <= 64 * 2.0 ** -24 * weights).all()
    _same(r.groups, group_ref(experts, E, k))


def test_route_infinities():
    logits = torch.tensor([[1.0, torch.inf, 2.0, torch.inf], [-torch.inf, -3e38, torch.nan, 3e38]], device="cuda")
    r = ops.moe_route(logits, 3)
    assert r.experts.tolist() == [[1, 3, 2], [3, 1, -1]]
    assert r.weights.tolist() == [[0.5, 0.5, 0.0], [1.0, 0.0, 0.0]]


@pytest.fixture
def form():
    def force(v):
        _lib.check("sfb200_debug_force_grouped", _lib.lib().sfb200_debug_force_grouped(v))
    yield force
    force(0)


def _weights(g, E, N, K, dt):
    w = randn(g, E, N, K, dtype=dt, scale=0.05)
    return ops.prune_compress_24(w.view(E * N, K), want_values=False, want_meta=False, want_pruned=True)["pruned"].view(E, N, K)


SIZES = [[0, 5, 0, 33], [241, 1, 0, 130], [16, 64, 65, 480], [0, 0, 0, 0], [0, 0, 700, 0]]
FORMS = [32, 64, 1128, 1240, 2128, 2240]


def _reference(x, w, sizes, bias):
    """Rows in the order of the experts: products, and what 32-bit sums of K terms may be off by (a rounding per term)."""
    y, slack, at = [], [], 0
    for e, n in enumerate(sizes):
        xe, we = x[at:at + n].double(), w[e].double()
        y.append(xe @ we.t() + (0 if bias is None else bias[e].double()))
        slack.append((xe.abs() @ we.abs().t() + (0 if bias is None else bias[e].double().abs())) * x.shape[1] * 2.0 ** -24)
        at += n
    return torch.cat(y), torch.cat(slack)


@pytest.mark.parametrize("variant", FORMS + [10000 + v for v in FORMS])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dt,N,K", [("bf16", 328, 192), ("f16", 640, 448)])
def test_grouped_store(form, variant, sizes, dt, N, K):
    gather, E, S = variant >= 10000, len(sizes), sum(sizes)
    g = gen(variant + S + N)
    w, bias = _weights(g, E, N, K, DT[dt]), randn(g, E, N, dtype=DT[dt])
    cw = ops.compress_experts(w)
    ids = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(sizes, device="cuda"))
    spare = torch.full((9,), -1, device="cuda")                       # entries of no expert: rows behind the last group
    perm = torch.randperm(S + 9, generator=g, device="cuda")
    groups = ops.group_rows(torch.cat([ids, spare])[perm] if gather else torch.cat([ids, spare]), E)
    x = randn(g, S + 9, K, dtype=DT[dt])
    if gather:
        x[(groups.slots < 0)] = torch.nan                             # read by no expert
    out = torch.full((S + 9, N + 8), 7.0, dtype=DT[dt], device="cuda")[:, :N]
    form(variant)
    ops.grouped_sparse_gemm(x, cw, groups, bias=bias, gather=gather, out=out)
    assert ops.device_status() == 0
    rows = groups.rows[:S].long()
    ref, slack = _reference(x[rows] if gather else x[:S], w, sizes, bias)
    close(out[:S], ref, slack)
    assert (out[S:] == 7).all()                                       # left as they were


@pytest.mark.parametrize("variant", FORMS + [10000 + v for v in FORMS])
@pytest.mark.parametrize("sizes", SIZES[:3])
@pytest.mark.parametrize("dt,I,K,biased", [("bf16", 176, 192, True), ("f16", 336, 576, False)])
def test_grouped_swiglu(form, variant, sizes, dt, I, K, biased):
    gather, E, S = variant >= 10000, len(sizes), sum(sizes)
    g = gen(variant + S + I)
    wg, wu = (_weights(g, E, I, K, DT[dt]) for _ in range(2))
    bg, bu = (randn(g, E, I, dtype=DT[dt]) if biased else None for _ in range(2))
    cw = ops.compress_gate_up_experts(wg, wu)
    ids = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(sizes, device="cuda"))
    groups = ops.group_rows(ids[torch.randperm(S, generator=g, device="cuda")] if gather else ids, E)
    x = randn(g, S, K, dtype=DT[dt])
    form(variant)
    out = ops.grouped_sparse_gemm_swiglu(x, cw, groups, gather=gather, gate_bias=bg, up_bias=bu)
    assert ops.device_status() == 0
    xr = x[groups.rows.long()] if gather else x
    (gate, gs), (up, us) = _reference(xr, wg, sizes, bg), _reference(xr, wu, sizes, bu)
    silu = gate * torch.sigmoid(gate)
    # silu' <= 1.1; the fast exponential and division are within 2^-20 at these arguments
    close(out, silu * up, 1.1 * gs * up.abs() + silu.abs() * us + gs * us + 2.0 ** -18 * (silu * up).abs())


@pytest.mark.parametrize("per_expert", [0.2, 3, 60, 130])
@pytest.mark.parametrize("gather", [False, True])
def test_many_experts(per_expert, gather):
    """1024 experts: whatever form the plan names, its tables fit."""
    E, N, K = 1024, 72, 64
    g = gen(int(per_expert * 10))
    w = _weights(g, E, N, K, torch.bfloat16)
    ids = torch.randint(0, E, (int(E * per_expert),), generator=g, device="cuda")
    groups = ops.group_rows(ids, E)
    x = randn(g, ids.numel(), K, dtype=torch.bfloat16)
    y = ops.grouped_sparse_gemm(x, ops.compress_experts(w), groups, gather=gather)
    assert ops.device_status() == 0
    rows, sizes = groups.rows.long(), groups.offsets.diff().tolist()
    close(y, *_reference(x[rows] if gather else x, w, sizes, None))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_grouped_activations(act):
    g = gen(5)
    w = _weights(g, 3, 136, 128, torch.float16)
    x = randn(g, 40, 128, dtype=torch.float16)
    sizes = [13, 0, 27]
    groups = ops.group_rows(torch.repeat_interleave(torch.arange(3), torch.tensor(sizes)).cuda(), 3)
    ref, slack = _reference(x, w, sizes, None)
    f = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act]
    close(ops.grouped_sparse_gemm(x, ops.compress_experts(w), groups, act=act), f(ref), 1.2 * slack + 2.0 ** -18 * ref.abs())


def test_grouped_strided_rows_and_one_expert():
    g = gen(9)
    w = _weights(g, 1, 264, 320, torch.bfloat16)
    cw = ops.compress_experts(w)
    for rows in (1, 5):
        for x in (randn(g, rows, 640, dtype=torch.bfloat16)[:, 320:], randn(g, rows, 325, dtype=torch.bfloat16)[:, 5:], randn(g, 320, rows, dtype=torch.bfloat16).t()):
            y = ops.grouped_sparse_gemm(x, cw, ops.group_rows(torch.zeros(rows, dtype=torch.int32, device="cuda"), 1))
            close(y, *_reference(x, w, [rows], None))


def test_grouped_offsets_out_of_range_stay_inside():
    """Offsets that no grouping makes (too large, descending) touch nothing outside the result."""
    g = gen(11)
    cw = ops.compress_experts(_weights(g, 3, 128, 128, torch.float16))
    x = randn(g, 32, 128, dtype=torch.float16)
    out = torch.full((40, 128), 7.0, dtype=torch.float16, device="cuda")
    for off in ([0, 500, 1000, 4000], [0, 20, 10, 30], [-5, 8, 16, 2 ** 31 - 1]):
        groups = ops.RowGroups(torch.tensor(off, dtype=torch.int32, device="cuda"), torch.zeros(32, dtype=torch.int32, device="cuda"), None, 3)
        ops.grouped_sparse_gemm(x, cw, groups, out=out[:32])
        ops.grouped_sparse_gemm(x, cw, groups, out=out[:32], gather=True)
        assert ops.device_status() == 0 and (out[32:] == 7).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("n,k,H", [(1, 1, 1), (3, 2, 8), (65, 6, 2048), (200, 8, 1707), (33, 3, 96), (1000, 5, 24)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(dt, n, k, H, residual):
    g = gen(n + H)
    rows = n * k
    y = randn(g, rows + 2, H + 8, dtype=DT[dt])[:, :H]
    slots = torch.randperm(rows, generator=g, device="cuda").to(torch.int32).view(n, k)
    if n > 2:
        slots[1] = -1                                           # a token of no expert
        slots[0, 0] = rows + 2                                  # outside y
    used = torch.zeros(rows + 2, dtype=torch.bool, device="cuda")
    live = (slots >= 0) & (slots < rows + 2)
    used[slots[live].long()] = True
    y[~used] = torch.nan
    weights = torch.rand(n, k, generator=g, device="cuda")
    res = randn(g, n, H, dtype=DT[dt]) if residual else None
    terms = torch.where(live.unsqueeze(2), weights.double().unsqueeze(2) * y[slots.clamp(0, rows + 1).long()].double(), 0.0)
    ref, size = terms.sum(1), terms.abs().sum(1)
    if residual:
        ref, size = ref + res.double(), size + res.double().abs()
    got = ops.moe_combine(y, slots, weights, residual=res)
    close(got, ref, (k + 1) * 2.0 ** -24 * size)
    if residual:
        assert torch.equal(ops.moe_combine(y, slots, weights, residual=res, out=res), got)


def test_refusals():
    g = gen(1)
    w = _weights(g, 2, 128, 128, torch.float16)
    cw, x = ops.compress_experts(w), randn(g, 6, 128, dtype=torch.float16)
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    groups = ops.group_rows(ids, 2)
    y = randn(g, 6, 16, dtype=torch.float16)
    s, wt = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    logits = randn(g, 4, 8)
    bad = [
        lambda: ops.group_rows(ids.float(), 2), lambda: ops.group_rows(ids, 0), lambda: ops.group_rows(ids, 1025), lambda: ops.group_rows(ids, 2, per_row=4),
        lambda: ops.moe_route(logits.double(), 2), lambda: ops.moe_route(logits, 0), lambda: ops.moe_route(logits, 9), lambda: ops.moe_route(logits[0], 2),
        lambda: ops.moe_route(randn(g, 2, 1025), 2),
        lambda: ops.compress_experts(w[0]), lambda: ops.compress_experts(w[:, :, :96]), lambda: ops.compress_experts(w.float()),
        lambda: ops.compress_gate_up_experts(w[:, :8], w[:, :8]), lambda: ops.compress_gate_up_experts(w, w[:1]),
        lambda: ops.grouped_sparse_gemm(x[:, :64], cw, groups), lambda: ops.grouped_sparse_gemm(x.bfloat16(), cw, groups),
        lambda: ops.grouped_sparse_gemm(x, cw, ops.group_rows(ids, 3)), lambda: ops.grouped_sparse_gemm(x[:5], cw, groups),
        lambda: ops.grouped_sparse_gemm(x, cw, ops.group_rows(ids, 2, per_row=2), gather=True),
        lambda: ops.grouped_sparse_gemm(x, cw, groups, act="tanh"), lambda: ops.grouped_sparse_gemm(x, cw, groups, bias=x[0]),
        lambda: ops.grouped_sparse_gemm(x, cw, groups, out=x), lambda: ops.grouped_sparse_gemm(x, cw, groups, out=x.float()),
        lambda: ops.grouped_sparse_gemm_swiglu(x, cw, groups), lambda: ops.grouped_sparse_gemm(x, ops.compress_gate_up_experts(w, w), groups),
        lambda: ops.moe_combine(y, s.long(), wt), lambda: ops.moe_combine(y, s, wt.half()), lambda: ops.moe_combine(y, s, wt[:2]),
        lambda: ops.moe_combine(y, s, wt, residual=y), lambda: ops.moe_combine(y, s, wt, out=y[:3]), lambda: ops.moe_combine(y.float(), s, wt),
        lambda: ops.moe_combine(y.cpu(), s, wt), lambda: ops.moe_combine(y, s.cpu(), wt),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
