"""Low-rank adapters of many requests beside a shared projection, against a 64-bit reference."""
import pytest
import torch

from sparseflow_b200 import ops
from sparseflow_b200.nn import SparseFlowLinear, SparseFlowPolicy

from .operator_refs import DT, close, gen, randn

pytestmark = pytest.mark.gpu


def _reference(x, y, a, b, scales, ids):
    """Every sum of K (and then rank) terms may be off by a rounding per term; u enters the second product with 2 half steps of its type less than exact,
    squared."""
    lost = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}[x.dtype]
    ref, slack = y.double().clone(), y.double().abs() * 2.0 ** -24
    for i in range(a.shape[0]):
        t = ids == i
        if t.any():
            s, xd, ad, bd = scales[i].double(), x[t].double(), a[i].double(), b[i].double()
            ref[t] += s * (xd @ ad.t()) @ bd.t()
            u = s.abs() * (xd.abs() @ ad.abs().t())
            slack[t] += u @ bd.abs().t() * (x.shape[1] + a.shape[1] + 4) * 2.0 ** -24 + (s * (xd @ ad.t())).abs() @ bd.abs().t() * lost
    return ref, slack


def _case(g, n, A, r, K, N, dt, ids=None):
    ids = torch.randint(-1, A, (n,), generator=g, device="cuda") if ids is None else ids.cuda()
    return (randn(g, n, K, dtype=dt), randn(g, n, N, dtype=dt), randn(g, A, r, K, dtype=dt, scale=K ** -0.5), randn(g, A, N, r, dtype=dt),
            0.5 + torch.rand(A, generator=g, device="cuda"), ids)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("r", [1, 8, 16, 24, 64, 100, 128])
@pytest.mark.parametrize("n,A,K,N", [(1, 1, 8, 8), (5, 3, 72, 40), (48, 64, 1000, 136), (200, 3, 576, 264), (700, 2, 4104, 72), (300, 300, 128, 64)])
def test_ranks_and_sizes(dt, r, n, A, K, N):
    x, y, a, b, s, ids = _case(gen(n + r + K), n, A, r, K, N, DT[dt])
    bank, groups = ops.LoraBank(a, b, s), ops.group_rows(ids, A)
    out = ops.lora_add(y, x, bank, groups)
    close(out, *_reference(x, y, a, b, s, ids))
    assert torch.equal(out[ids < 0], y[ids < 0])
    again = y.clone()
    assert ops.lora_add(again, x, bank, groups, out=again) is again and torch.equal(again, out)      # in place, the same bits


@pytest.mark.parametrize("ids", [torch.full((40,), -1), torch.full((40,), 2), torch.arange(40) % 3, torch.zeros(0, dtype=torch.long), torch.arange(500) // 250])
def test_groupings(ids):
    x, y, a, b, s, ids = _case(gen(len(ids)), len(ids), 3, 16, 256, 96, torch.bfloat16, ids)
    close(ops.lora_add(y, x, ops.LoraBank(a, b, s), ops.group_rows(ids, 3)), *_reference(x, y, a, b, s, ids))


@pytest.mark.parametrize("n,A", [(9, 4), (400, 2)])
def test_strides(n, A):
    g = gen(n)
    x, y, a, b, s, ids = _case(g, n, A, 16, 256, 96, torch.float16)
    bank, groups = ops.LoraBank(a, b, s), ops.group_rows(ids, A)
    ref = ops.lora_add(y, x, bank, groups)
    wide = torch.zeros(n, 512, dtype=torch.float16, device="cuda")
    for at, width in ((256, 512), (3, 300)):                                # rows of a wider tensor, aligned and not
        xw = torch.zeros(n, width, dtype=torch.float16, device="cuda")
        xw[:, at:at + 256] = x
        yw = torch.full((n, width), 3.0, dtype=torch.float16, device="cuda")
        yw[:, at:at + 96] = y
        assert torch.equal(ops.lora_add(yw[:, at:at + 96], xw[:, at:at + 256], bank, groups), ref)
        ops.lora_add(yw[:, at:at + 96], xw[:, at:at + 256], bank, groups, out=yw[:, at:at + 96])
        assert torch.equal(yw[:, at:at + 96], ref) and (yw[:, at + 96:] == 3).all() and (yw[:, :at] == 3).all()
    out = wide[:, 8:104]
    assert torch.equal(ops.lora_add(y, x, bank, groups, out=out), ref) and (wide[:, :8] == 0).all()


def test_more_rows_than_a_grid_dimension():
    """2.2 million rows (tiles and copies above 65535), in place and not; compared with the same rows in two calls."""
    n, g = 2_200_000, gen(12)
    x, y, a, b, s, ids = _case(g, n, 2, 8, 8, 8, torch.bfloat16)
    bank = ops.LoraBank(a, b, s)
    out = ops.lora_add(y, x, bank, ops.group_rows(ids, 2))
    for part in (slice(0, 3000), slice(n - 3000, n)):
        close(out[part], *_reference(x[part], y[part], a, b, s, ids[part]))
    assert torch.equal(out[ids < 0], y[ids < 0])
    assert torch.equal(ops.lora_add(y, x, bank, ops.group_rows(ids, 2), out=y), out)


def test_large_and_small_products_of_f16():
    """u beyond the range of f16 and far below it: the row is scaled by a power of two."""
    g = gen(2)
    x, y, a, b, s, ids = _case(g, 6, 1, 16, 512, 64, torch.float16, torch.zeros(6, dtype=torch.long))
    for sa, sb, scale in ((2.0 ** 17, 2.0 ** -17, 1.0), (2.0 ** -8, 2.0 ** 10, 2.0 ** -12)):
        aa, bb, ss, y0 = (a.float() * sa).half(), (b.float() * sb).half(), torch.tensor([scale], device="cuda"), torch.zeros_like(y)
        close(ops.lora_add(y0, x, ops.LoraBank(aa, bb, ss), ops.group_rows(ids, 1)), *_reference(x, y0, aa, bb, ss, ids))


def test_infinities_stay_in_their_row():
    g = gen(6)
    for n in (8, 200):
        x, y, a, b, s, ids = _case(g, n, 1, 16, 256, 64, torch.bfloat16, torch.zeros(n, dtype=torch.long))
        clean = ops.lora_add(y, x, ops.LoraBank(a, b, s), ops.group_rows(ids, 1))
        x[3, 9], x[5, 200] = torch.inf, torch.nan
        out = ops.lora_add(y, x, ops.LoraBank(a, b, s), ops.group_rows(ids, 1))
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        keep[[3, 5]] = False
        assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[5]).all() and not torch.isfinite(out[3]).any()


def test_bank_of_mixed_ranks():
    g = gen(7)
    pairs = [(randn(g, r, 128, dtype=torch.bfloat16), randn(g, 48, r, dtype=torch.bfloat16)) for r in (4, 16, 9)]
    bank = ops.LoraBank.from_adapters(pairs, scales=2.0)
    ids = torch.tensor([2, 0, 1, 1, 2, -1], device="cuda")
    x, y = randn(g, 6, 128, dtype=torch.bfloat16), randn(g, 6, 48, dtype=torch.bfloat16)
    pad = torch.nn.functional.pad
    a = torch.stack([pad(A, (0, 0, 0, 16 - A.shape[0])) for A, _ in pairs])
    b = torch.stack([pad(B, (0, 16 - B.shape[1])) for _, B in pairs])
    close(ops.lora_add(y, x, bank, ops.group_rows(ids, 3)), *_reference(x, y, a, b, torch.full((3,), 2.0, device="cuda"), ids))


@pytest.mark.parametrize("sparse", [True, False])
def test_linear_with_adapters(sparse):
    g = gen(8)
    w = randn(g, 192, 256, dtype=torch.bfloat16, scale=0.05)
    policy = SparseFlowPolicy(min_M_default=0 if sparse else 10 ** 9)
    lin = SparseFlowLinear(w, None, policy=policy, op_name="shared")
    x = randn(g, 2, 7, 256, dtype=torch.bfloat16)
    base = lin(x)
    ids = torch.tensor([0, 0, -1, 1, 1, 1, 0, 2, -1, 2, 2, 0, 1, 0], device="cuda")
    a, b = randn(g, 3, 16, 256, dtype=torch.bfloat16, scale=0.06), randn(g, 3, 192, 16, dtype=torch.bfloat16)
    groups = ops.group_rows(ids, 3)
    with pytest.raises(ValueError):
        lin(x, groups)
    bank = ops.LoraBank(a, b)
    lin.set_adapters(bank)
    want = ops.lora_add(base.view(14, 192), x.view(14, 256), bank, groups)
    assert torch.equal(lin(x, groups).view(14, 192), want) and torch.equal(lin(x), base)
    assert (lin._sparse_count > 0) == sparse
    with pytest.raises(ValueError):
        lin.set_adapters(ops.LoraBank(a.half(), b.half()))
    with pytest.raises(ValueError):
        lin.set_adapters(ops.LoraBank(b, a))


def test_refusals():
    x, y, a, b, s, ids = _case(gen(9), 6, 2, 16, 64, 32, torch.bfloat16)
    bank, groups = ops.LoraBank(a, b, s), ops.group_rows(ids, 2)
    square = ops.LoraBank(randn(gen(1), 2, 8, 64, dtype=torch.bfloat16), randn(gen(1), 2, 64, 8, dtype=torch.bfloat16))
    bad = [
        lambda: ops.LoraBank(a, b[:1]), lambda: ops.LoraBank(a, b.half()), lambda: ops.LoraBank(a.float(), b.float()), lambda: ops.LoraBank(a, b, s[:1]),
        lambda: ops.LoraBank(a[:, :, :60], b), lambda: ops.LoraBank(a.cpu(), b.cpu()),
        lambda: ops.LoraBank(torch.zeros(1, 129, 64, dtype=torch.half, device="cuda"), torch.zeros(1, 64, 129, dtype=torch.half, device="cuda")),
        lambda: ops.lora_add(y, x[:5], bank, groups), lambda: ops.lora_add(y[:, :24], x, bank, groups), lambda: ops.lora_add(y.half(), x, bank, groups),
        lambda: ops.lora_add(y, x, bank, ops.group_rows(ids, 3)), lambda: ops.lora_add(y, x, bank, ops.group_rows(ids, 2, per_row=2)),
        lambda: ops.lora_add(y.cpu(), x, bank, groups), lambda: ops.lora_add(y, x, bank, groups, out=y[:5]), lambda: ops.lora_add(y, x, bank, groups, out=y.float()),
        lambda: ops.lora_add(x, x, square, groups, out=x.view(-1)[:384].view(6, 64)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
