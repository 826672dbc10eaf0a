"""What DraftBlock refuses without a GPU: the steps of a block that has no 8-bit cache, or no vocabulary."""
import pytest
import torch

from fp6_marlin_b200.draft_step import DraftBlock


def test_steps_that_a_block_has_not():
    block = DraftBlock(hidden=256, inter=256, heads=2, kv_heads=2, sequences=2, tokens=3, pages=4, quant_cols=0, device="cpu")
    keys = torch.zeros((2, 3, 2, 128), dtype=torch.float16)
    accepted, counts = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    table, lengths = torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="accept"):
        block.commit(keys, keys, accepted, counts, table, lengths)
    assert not lengths.any()
    with pytest.raises(ValueError, match="vocab"):
        block.choose(torch.zeros((6, 256), dtype=torch.float16), accepted.long(), torch.ones((2, 3), dtype=torch.int64), torch.zeros((2, 3)))
