"""DraftBlock.commit where some accepted tokens have no place: lengths count those that stand in the cache."""
import pytest
import torch

import fp6_marlin_b200 as fm
from test_gpu_draft_step_fp8 import _block

pytestmark = pytest.mark.gpu


def test_lengths_count_what_was_written():
    block = _block(8, 2, 4, sequences=5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    keys, values = (torch.randn((5, 4, 2, 128), generator=gen, device="cuda").half() for _ in range(2))
    table = torch.randperm(128, generator=gen, device="cuda")[:15].view(5, 3).int()
    table[2, 1] = -1                                               # a page that does not exist: tokens 16 .. 31
    table[3, 2] = 128
    #             room       one place          a page missing    likewise, at its end   a number that no token has
    lengths = torch.tensor([10, 47, 14, 30, 0], dtype=torch.int32, device="cuda")
    accepted = torch.tensor([[0, 1, 2, -1], [0, 2, 3, -1], [0, 1, 2, 3], [0, 1, 3, -1], [0, 4, 2, -1]], dtype=torch.int32, device="cuda")
    counts = torch.tensor([3, 3, 4, 3, 3], dtype=torch.int32, device="cuda")
    block.commit(keys, values, accepted, counts, table, lengths)
    assert fm.device_status() == 4 and lengths.dtype == torch.int32
    assert lengths.tolist() == [13, 48, 16, 32, 1]
    block.commit(keys, values, accepted, counts, table[:, :0], lengths)      # no place at all
    assert fm.device_status() == 4 and lengths.tolist() == [13, 48, 16, 32, 1]
    lengths.copy_(torch.tensor([0, 1, 2, 3, 4], device="cuda"))
    table[2, 1], table[3, 2], accepted[4, 1] = 90, 91, 1
    block.commit(keys, values, accepted, torch.zeros_like(counts), table, lengths)
    assert lengths.tolist() == [0, 1, 2, 3, 4]
    block.commit(keys, values, accepted[:, :2].contiguous(), counts.clamp(max=2), table, lengths)
    assert fm.device_status() == 0 and lengths.tolist() == [2, 3, 4, 5, 6]
    block.commit(keys, values, accepted, counts, table, lengths)
    assert fm.device_status() == 0 and lengths.tolist() == [5, 6, 8, 8, 9]
