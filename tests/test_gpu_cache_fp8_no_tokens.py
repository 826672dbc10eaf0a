"""write_cache_fp8 where there are no new tokens to take from: a list of entries that name none is nothing to do, one that names one is reported."""
import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_entries_without_tokens(dtype):
    cache, table, lengths = fm.make_cache_fp8(6, 16, 2, 64), torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3), torch.tensor([5, 40], dtype=torch.int32, device="cuda")
    none = torch.zeros((2, 0, 2, 64), dtype=dtype, device="cuda")
    entries = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    counts = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    fm.write_cache_fp8(none, none, *cache, table, lengths)
    fm.write_cache_fp8(none, none, *cache, table, lengths, tokens=entries)
    fm.write_cache_fp8(none, none, *cache, table, lengths, tokens=entries, counts=counts)
    assert fm.device_status() == 0
    entries[1, 2] = 0                                              # behind the sequence's count
    fm.write_cache_fp8(none, none, *cache, table, lengths, tokens=entries, counts=counts)
    assert fm.device_status() == 0
    fm.write_cache_fp8(none, none, *cache, table, lengths, tokens=entries)
    assert fm.device_status() == 4
    assert not any(c.view(torch.uint8).any() for c in cache[:2]) and all((c == 127).all() for c in cache[2:])
