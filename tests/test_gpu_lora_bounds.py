"""A grouping that no call of the library makes (written by hand, or overwritten) reads and writes nothing outside the batch."""
import pytest
import torch

from sparseflow_b200 import ops

from .operator_refs import gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,A", [(9, 4), (400, 3)])      # tiles of 16 rows, of 128 rows
@pytest.mark.parametrize("rank", [16, 64])
def test_offsets_and_rows_out_of_range(n, A, rank):
    g, K, N, dt = gen(n + rank), 256, 96, torch.bfloat16
    x, y = randn(g, n, K, dtype=dt), randn(g, n, N, dtype=dt)
    bank = ops.LoraBank(randn(g, A, rank, K, dtype=dt), randn(g, A, N, rank, dtype=dt))
    good = ops.group_rows(torch.arange(n, device="cuda") % A, A)
    ref = ops.lora_add(y, x, bank, good)
    buf = torch.full((n + 16, N), 7.0, dtype=dt, device="cuda")
    out = buf[8:n + 8]

    def run(offsets, rows):
        groups = ops.RowGroups(torch.tensor(offsets, dtype=torch.int32, device="cuda"), rows, good.slots, A)
        ops.lora_add(y, x, bank, groups, out=out)
        assert ops.device_status() == 0 and (buf[:8] == 7).all() and (buf[n + 8:] == 7).all()

    last = 2 ** 31 - 1
    for off in ([0, 500, 1000, 4000, 5000], [0, n, n // 2, 3, last], [-5, 3, -7, 6, last], [last] * 5, [-2 ** 31, last, -1, last, 0]):
        run(off[:A + 1], good.rows)
    rows = good.rows.clone()
    rows[0], rows[n // 2], rows[n - 1] = n, -5, last
    run(good.offsets.tolist(), rows)
    kept = torch.ones(n, dtype=torch.bool, device="cuda")
    kept[good.rows[[0, n // 2, n - 1]].long()] = False      # the other rows are what they are with a good grouping
    assert torch.equal(out[kept], ref[kept])
