"""The first call of the library in a process may be one that is captured: what it sets up on the device does not end the capture."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from sparseflow_b200 import ops
g = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
x, y, w = r(700, 4096), r(700, 4096), r(4096)
ids = torch.arange(700, device="cuda", dtype=torch.int32) % 3
bank = ops.LoraBank(r(3, 16, 4096), r(3, 4096, 16))
slots, weights = torch.randint(0, 700, (50, 4), generator=g, device="cuda").int(), torch.rand(50, 4, generator=g, device="cuda")
def route():
    t = ops.moe_route(x[:, :64], 4)
    return t.weights, t.experts, t.groups.offsets, t.groups.rows, t.groups.slots
calls = {"norm": lambda: ops.block_norm(x, y, weight=w, post_weight=w), "route": route, "combine": lambda: (ops.moe_combine(x, slots, weights),),
         "adapters": lambda: (ops.lora_add(y, x, bank, ops.group_rows(ids, 3)),), "silu": lambda: (ops.silu_mul(x, y),)}
call = calls["CALL"]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, call())) and ops.device_status() == 0
print("the same")
"""


@pytest.mark.parametrize("call", ["norm", "route", "combine", "adapters", "silu"])
def test_first_call(call):
    r = subprocess.run([sys.executable, "-c", PROGRAM.replace("CALL", call)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]
