"""The operators around the FFN from several threads at once, each on its own stream: the results of one thread after the other."""
import threading

import pytest
import torch

from sparseflow_b200 import ops
from sparseflow_b200.nn import SparseFlowMoE

from .operator_refs import gen, randn

pytestmark = pytest.mark.gpu


def _work(seed):
    g, dt = gen(seed), torch.bfloat16
    E, H, I, n = 6, 512, 704, 40 + 500 * (seed % 3)
    moe = SparseFlowMoE(randn(g, E, H, scale=0.2), randn(g, E, I, H, dtype=dt, scale=0.05), randn(g, E, I, H, dtype=dt, scale=0.05),
                        randn(g, E, H, I, dtype=dt, scale=0.05), 2)
    x, y, w = randn(g, n, H, dtype=dt), randn(g, n, H, dtype=dt), randn(g, H, dtype=dt)
    bank = ops.LoraBank(randn(g, 3, 16, H, dtype=dt, scale=0.05), randn(g, 3, H, 16, dtype=dt))
    ids = torch.randint(-1, 3, (n,), generator=g, device="cuda")

    def run():
        r, h = ops.block_norm(x, y, weight=w, post_weight=w)
        out = moe(h, residual=r)
        return ops.lora_add(out, h, bank, ops.group_rows(ids, 3))

    return run


def test_threads():
    work = [_work(s) for s in range(6)]
    want = [run() for run in work]
    torch.cuda.synchronize()
    wrong = []

    def body(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got = work[i]()
                    stream.synchronize()
                    if not torch.equal(got, want[i]):
                        wrong.append(i)
        except Exception as e:      # noqa: BLE001: a thread's exception is not the test's
            wrong.append((i, e))

    threads = [threading.Thread(target=body, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and ops.device_status() == 0
