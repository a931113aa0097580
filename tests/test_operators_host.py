"""What the operators around the FFN decide and refuse on the host."""
import pytest
import torch

from sparseflow_b200 import ops


def test_calls_refuse_cpu_tensors():
    x, ids = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32)
    groups = ops.RowGroups(torch.zeros(3, dtype=torch.int32), ids, ids, 2)
    bank = object.__new__(ops.LoraBank)
    cw = ops.CompressedExperts(x, x, 2, 64, 64)
    for call in (lambda: ops.group_rows(ids, 2), lambda: ops.moe_route(x, 2), lambda: ops.moe_route(logits=x, top_k=2), lambda: ops.compress_experts(x[None]),
                 lambda: ops.compress_gate_up_experts(x[None], x[None]), lambda: ops.grouped_sparse_gemm(x, cw, groups),
                 lambda: ops.grouped_sparse_gemm_swiglu(x, cw, groups), lambda: ops.moe_combine(x, ids.view(2, 2), torch.ones(2, 2)),
                 lambda: ops.block_norm(x, weight=x[0]), lambda: ops.LoraBank(x[None], x[None]), lambda: ops.lora_add(x, x, bank, groups)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_memory_shared_with_the_result():
    t = torch.zeros(8, 16)
    ops._check_apart(t[:, :8], t[4:, :8].clone(), "x")
    ops._check_apart(t[:4], t[4:], "x")
    ops._check_apart(t, t, "y", same=True)
    ops._check_apart(t[:0], t, "x")
    for out, other, same in ((t, t, False), (t[1:], t[:-1], True), (t[:, 8:], t[:, :8], False), (t[:4], t[3:7], True), (t.view(-1)[:64].view(4, 16), t.view(-1)[8:72].view(4, 16), True)):
        with pytest.raises(ValueError):
            ops._check_apart(out, other, "x", same=same)


FORMS = {32, 64, 1128, 1240, 2128, 2240}


def test_plan_of_grouped_products(lib):
    """Every size gets a form of the kernel; few tokens per expert the small tiles, many the pairs; rows are copied only where they are gathered."""
    for total in (1, 7, 100, 2000, 50000, 1 << 24):
        for experts in (1, 2, 8, 100, 1024):
            for N, K in ((8, 64), (1000, 512), (4096, 11008), (22016, 4096)):
                for sms in (16, 148):
                    assert lib.sfb200_debug_plan_grouped(total, experts, N, K, 0, sms) in FORMS
                    assert lib.sfb200_debug_plan_grouped(total, experts, N, K, 1, sms) % 10000 in FORMS
    assert lib.sfb200_debug_plan_grouped(16, 8, 22016, 4096, 0, 148) in (32, 64)
    assert lib.sfb200_debug_plan_grouped(4096, 8, 22016, 4096, 0, 148) >= 1000
    assert lib.sfb200_debug_plan_grouped(8192, 8, 22016, 4096, 1, 148) >= 10000
    assert lib.sfb200_debug_plan_grouped(16, 8, 22016, 4096, 1, 148) < 10000
    assert lib.sfb200_debug_plan_grouped(0, 8, 22016, 4096, 1, 148) == 0


def test_workspace_sizes(lib):
    assert lib.sfb200_group_workspace_bytes(128) == 128 * 128 * 4 and lib.sfb200_group_workspace_bytes(0) == 0
    assert lib.sfb200_lora_workspace_bytes(10, 16) == 10 * 17 * 4 and lib.sfb200_lora_workspace_bytes(0, 16) == 0


def test_calls_without_a_device_return_an_error(lib):
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    assert lib.sfb200_group_rows(None, 0, 1, 1, None, None, None, None, None) != 0
    assert lib.sfb200_moe_combine(None, 8, 0, None, None, None, 0, None, 8, 0, 1, 8, 0, None) != 0
    assert lib.sfb200_grouped_scratch_bytes(100, 8, 64, 64) == 0


def test_counts_beyond_32_bits_are_refused():
    huge = torch.empty(1, device="meta", dtype=torch.float16).expand(2 ** 31, 1)
    with pytest.raises(ValueError, match="32-bit"):
        ops._rows2d(huge, "x")


def test_direct_calls_convert_like_the_c_abi(lib):
    """The module beside the library: the same functions, whole ranges checked, wrong counts and types refused."""
    from sparseflow_b200 import _lib
    calls = _lib.calls()
    names = [n for n in dir(calls) if n.startswith("sfb200_")]
    assert len(names) == 10
    for n in names:
        arity = len(getattr(lib, n).argtypes)
        for count in (arity - 1, arity + 1):
            with pytest.raises(TypeError, match=f"expected {arity} arguments"):
                getattr(calls, n)(*[0] * count)
    for args in ((10, 16), (2 ** 31 - 1, 128)):
        assert calls.sfb200_lora_workspace_bytes(*args) == lib.sfb200_lora_workspace_bytes(*args)
    for n in (2 ** 31, -2 ** 31 - 1, 2 ** 70):
        with pytest.raises(OverflowError):
            calls.sfb200_group_workspace_bytes(n)
    with pytest.raises(TypeError):
        calls.sfb200_group_workspace_bytes("8")


def test_layouts_that_are_not_only_router_and_experts_are_refused():
    from torch import nn
    from sparseflow_b200.nn.sparseflow_moe import make_sparseflow_moe

    def expert(act=None):
        m = nn.Module()
        m.gate_proj, m.up_proj, m.down_proj = nn.Linear(64, 64, bias=False), nn.Linear(64, 64, bias=False), nn.Linear(64, 64, bias=False)
        if act is not None:
            m.act_fn = act
        return m

    def block(**kw):
        m = nn.Module()
        m.gate, m.experts, m.top_k = nn.Linear(64, 2, bias=False), nn.ModuleList([expert(**kw) for _ in range(2)]), 1
        return m

    m = block()
    m.shared_expert = expert()
    with pytest.raises(RuntimeError, match="shared_expert"):
        make_sparseflow_moe(m)
    for act in (nn.GELU(), nn.functional.relu):
        with pytest.raises(RuntimeError, match="SiLU"):
            make_sparseflow_moe(block(act=act))
    for act in (None, nn.SiLU(), nn.functional.silu):
        with pytest.raises(ValueError, match="CUDA"):      # accepted: the weights are what is refused here
            make_sparseflow_moe(block(act=act))
