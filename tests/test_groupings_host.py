"""A grouping written by hand is looked at before a kernel reads through it."""
import pytest
import torch

from sparseflow_b200 import ops


def _int(n, dtype=torch.int32):
    return torch.zeros(n, dtype=dtype)


def test_hand_written_groupings():
    t = torch.zeros(1)
    ops._check_groups(t, ops.RowGroups(_int(4), _int(9), _int(9), 3), True)
    ops._check_groups(t, ops.RowGroups(_int(4), _int(9), None, 3), False)
    bad = [(_int(3), _int(9), _int(9)), (_int(5), _int(9), _int(9)), (_int(4), _int(9), _int(8)), (_int(4, torch.int64), _int(9), _int(9)),
           (_int(4), _int(9, torch.int64), _int(9)), (_int(4), _int(9), _int(9, torch.float32)), (_int(8)[::2], _int(9), _int(9)),
           (_int(4), _int(18)[::2], _int(9)), (_int(4).to("meta"), _int(9), _int(9)), (_int(4), _int(9).to("meta"), _int(9))]
    for offsets, rows, slots in bad:
        with pytest.raises(ValueError):
            ops._check_groups(t, ops.RowGroups(offsets, rows, slots, 3), True)


def test_groupings_made_here_are_not_looked_at_again():
    groups = ops.RowGroups(_int(4), _int(9), _int(9), 3, 1, True)
    assert groups == groups and "made_here" not in repr(groups)
    with pytest.raises(ValueError, match="CUDA"):      # but for their device
        ops._check_groups(torch.zeros(1), groups, True)
