"""The operators around the FFN as they are used together: a mixture of experts between block norms, captured and replayed, on other streams,
and the prefill command that runs them."""
import pytest
import torch
import torch.nn.functional as F

from sparseflow_b200 import ops, prefill_e2e
from sparseflow_b200.nn import SparseFlowBlockNorm, SparseFlowMoE, make_sparseflow_moe, replace_llama_mlp_module

from .operator_refs import HALF_STEP, gen, randn

pytestmark = pytest.mark.gpu


def _moe(g, E, H, I, top_k, dt, biased=False, router=torch.float32, **kw):
    prune = lambda w: ops.prune_compress_24(w.view(-1, w.shape[-1]), want_values=False, want_meta=False, want_pruned=True)["pruned"].view_as(w)  # noqa: E731
    gate, up, down = (prune(randn(g, *s, dtype=dt, scale=0.06)) for s in ((E, I, H), (E, I, H), (E, H, I)))
    b = [randn(g, E, n, dtype=dt) if biased else None for n in (I, I, H)]
    wr = randn(g, E, H, dtype=router, scale=0.2)
    return SparseFlowMoE(wr, gate, up, down, top_k, gate_bias=b[0], up_bias=b[1], down_bias=b[2], **kw), (gate, up, down, *b)


def _moe_ref(x, routing, w):
    gate, up, down, bg, bu, bd = (None if t is None else t.double() for t in w)
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    for t in range(x.shape[0]):
        for p, e in zip(routing.weights[t].double(), routing.experts[t].tolist()):
            if e < 0:
                continue
            g, u = gate[e] @ x[t].double(), up[e] @ x[t].double()
            if bg is not None:
                g, u = g + bg[e], u + bu[e]
            h = (g * torch.sigmoid(g) * u).to(x.dtype).double()      # hidden values are 16-bit
            y = down[e] @ h + (0 if bd is None else bd[e])
            out[t] += p * y
            size[t] += p * (y.abs() + down[e].abs() @ h.abs())
    return out, size


@pytest.mark.parametrize("n,E,k,biased,renorm", [(1, 4, 2, False, True), (37, 5, 3, True, True), (300, 3, 1, False, False)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_moe_layer(n, E, k, biased, renorm, dt):
    g = gen(n + E)
    m, w = _moe(g, E, 128, 192, k, dt, biased, renormalize=renorm)
    x = randn(g, n, 128, dtype=dt)
    res = randn(g, n, 128, dtype=dt)
    out = m(x, residual=res)
    ref, size = _moe_ref(x, m.route(x), w)
    # roundings: a hidden value may fall to its other neighbour (a step), a row of y and the result half a step
    assert ((out.double() - ref - res.double()).abs() <= 2 * HALF_STEP[dt] * (2 * size + res.double().abs()) + 2.0 ** -24).all()
    assert m(x[:0]).shape == (0, 128)
    with pytest.raises(ValueError):
        m(x[:, :64])


def _block(norm, moe, x, y):
    r, h = norm(x, y)
    return moe(h, residual=r)


def test_captured_replayed_and_on_other_streams():
    """norm -> router -> products -> sum in one graph; replays with other inputs, and with another grouping, equal eager calls."""
    g = gen(3)
    moe, _ = _moe(g, 8, 256, 320, 2, torch.bfloat16, router=torch.bfloat16)
    norm = SparseFlowBlockNorm(randn(g, 256, dtype=torch.bfloat16), post_weight=randn(g, 256, dtype=torch.bfloat16))
    xs = [(randn(g, 90, 256, dtype=torch.bfloat16), randn(g, 90, 256, dtype=torch.bfloat16)) for _ in range(4)]
    x, y = (t.clone() for t in xs[0])
    eager = [_block(norm, moe, *p) for p in xs]
    assert torch.equal(eager[0], _block(norm, moe, *xs[0]))          # the same bits again
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = _block(norm, moe, *xs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(beside, eager[1])
    graphs = []
    for _ in range(2):                                               # two graphs: each has its workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block(norm, moe, x, y)
        graphs.append((graph, out))
    for i in (2, 3, 1):
        x.copy_(xs[i][0])
        y.copy_(xs[i][1])
        for graph, out in graphs:
            graph.replay()
        assert all(torch.equal(out, eager[i]) for _, out in graphs)
    assert ops.device_status() == 0


def test_adapters_captured():
    g = gen(4)
    x, y = randn(g, 200, 512, dtype=torch.float16), randn(g, 200, 256, dtype=torch.float16)
    bank = ops.LoraBank(randn(g, 3, 16, 512, dtype=torch.float16, scale=0.05), randn(g, 3, 256, 16, dtype=torch.float16))
    ids = torch.randint(-1, 3, (200,), generator=g, device="cuda").to(torch.int32)
    call = lambda: ops.lora_add(y, x, bank, ops.group_rows(ids, 3))  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in (1, 2):
        ids.copy_(torch.randint(-1, 3, (200,), generator=gen(seed), device="cuda"))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, call())


def test_padding_changes_nothing():
    """Rows of padding (logits of -inf) cost no expert anything and come out as zero."""
    g = gen(5)
    moe, _ = _moe(g, 4, 128, 128, 2, torch.bfloat16)
    x = randn(g, 50, 128, dtype=torch.bfloat16)
    logits = F.linear(x.float(), moe.router_weight)
    logits[40:] = -torch.inf
    r = ops.moe_route(logits, 2)
    gu, down = moe._weights()
    y = ops.grouped_sparse_gemm(ops.grouped_sparse_gemm_swiglu(x, gu, r.groups, gather=True), down, r.groups)
    out = ops.moe_combine(y, r.groups.slots, r.weights)
    assert (out[40:] == 0).all() and torch.equal(out[:40], moe(x[:40]))


def test_from_module_and_surgery():
    torch.manual_seed(0)
    mlp = prefill_e2e.MoEMLP(128, 192, 4, 2, device="cuda", dtype=torch.bfloat16)
    for p in mlp.parameters():
        p.data.normal_(0, 0.06)
    for e in mlp.experts:
        for lin in (e.gate_proj, e.up_proj, e.down_proj):
            lin.weight.data.copy_(ops.prune_compress_24(lin.weight.data, want_values=False, want_meta=False, want_pruned=True)["pruned"])
    moe = make_sparseflow_moe(mlp)
    assert (moe.experts, moe.top_k, moe.renormalize) == (4, 2, True)
    x = randn(gen(6), 3, 11, 128, dtype=torch.bfloat16)
    with torch.no_grad():
        want = mlp(x).double()
    # the plain module rounds gate, up, their product, hidden and every expert's row to 8 bits: a few half steps of the largest
    assert (moe(x).double() - want).abs().max() <= 8 * 2.0 ** -8 * want.abs().max()
    layer = torch.nn.Module()
    layer.mlp = mlp
    model = torch.nn.Module()
    model.layers = torch.nn.ModuleList([layer])
    assert replace_llama_mlp_module(model, None) == 1 and isinstance(layer.mlp, SparseFlowMoE)
    assert torch.equal(layer.mlp(x), moe(x))
    with pytest.raises(RuntimeError):
        make_sparseflow_moe(layer)
    with pytest.raises(ValueError):
        SparseFlowMoE(moe.router_weight[:3], *(torch.zeros(4, 64, 64, dtype=torch.half, device="cuda") for _ in range(3)), top_k=2)


@pytest.mark.parametrize("experts", [0, 4])
def test_prefill_command(experts):
    r = prefill_e2e.run(layers=2, hidden=256, inter=512, heads=4, batch=1, seq=64, iters=1, warmup=1, experts=experts)
    assert r["mlp_layers_replaced"] == 2 and r["norms_fused"] == 5 and "fused_norms" in r["arms"]
    if not experts:      # with experts a rounding may send a token elsewhere
        # five norms, each read with three 8-bit roundings more or less (2^-8 a half step)
        assert r["fused_norms_max_err_over_max"] <= 15 * 2.0 ** -8


def _far(g, rows, cols, dtype, pitch=2 ** 28):
    """``rows`` rows of one buffer, so far from each other that element offsets pass 32 bits (the buffer is not written between them)."""
    buf = torch.empty((rows - 1) * pitch + cols, dtype=dtype, device="cuda")
    t = buf.as_strided((rows, cols), (pitch, 1))
    t.copy_(randn(g, rows, cols, dtype=dtype))
    return t


def test_offsets_beyond_32_bits():
    """Rows up to 3.2e9 elements from the first: the same results as of a dense copy, bit for bit."""
    g, n, H, dt = gen(11), 13, 256, torch.bfloat16
    x = _far(g, n, H, dt)
    dense = x.contiguous()
    ids = torch.arange(n, dtype=torch.int32, device="cuda") % 3
    groups = ops.group_rows(ids, 3)
    cw = ops.compress_experts(randn(g, 3, 128, H, dtype=dt))
    for gather in (False, True):
        assert torch.equal(ops.grouped_sparse_gemm(x, cw, groups, gather=gather), ops.grouped_sparse_gemm(dense, cw, groups, gather=gather))
    weight = randn(g, H, dtype=dt)
    for a, b in zip(ops.block_norm(x, dense, weight=weight), ops.block_norm(dense, dense, weight=weight)):
        assert torch.equal(a, b)
    slots, weights = torch.randint(0, n, (9, 4), generator=g, device="cuda").int(), torch.rand(9, 4, generator=g, device="cuda")
    assert torch.equal(ops.moe_combine(x, slots, weights), ops.moe_combine(dense, slots, weights))
    assert torch.equal(ops.moe_route(x, 4).experts, ops.moe_route(dense, 4).experts)
    bank = ops.LoraBank(randn(g, 3, 16, H, dtype=dt), randn(g, 3, H, 16, dtype=dt))
    ref = ops.lora_add(dense, dense, bank, groups)
    assert torch.equal(ops.lora_add(x, dense, bank, groups), ref) and torch.equal(ops.lora_add(dense, x, bank, groups), ref)
    ops.lora_add(x, dense, bank, groups, out=x)
    assert torch.equal(x.contiguous(), ref)
    assert ops.device_status() == 0


def test_norms_captured_together_on_two_streams():
    """Two graphs of norms whose blocks stay, replayed at the same time on two streams with changed inputs: nothing is shared between them."""
    g, n, dt = gen(12), 2000, torch.bfloat16
    sets = []
    for H in (4096, 4099):
        x, y, w = randn(g, n, H), randn(g, n, H, dtype=dt), randn(g, H, dtype=dt)
        run = lambda x=x, y=y, w=w: ops.block_norm(x, y, weight=w, post_weight=w, kind="layer")  # noqa: E731
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        sets.append((x, y, run, graph, out, torch.cuda.Stream()))
    for _ in range(3):
        for x, y, *_rest in sets:
            x.copy_(randn(g, *x.shape))
            y.copy_(randn(g, *y.shape, dtype=dt))
        torch.cuda.synchronize()
        for *_rest, graph, out, stream in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for x, y, run, graph, out, stream in sets:
            for a, b in zip(out, run()):
                assert torch.equal(a, b)
