"""DraftBlock.accept on the CPU: where the keys and values of accepted tokens go."""
import pytest
import torch

from fp6_marlin_b200.draft_step import DraftBlock


def _block(pages=8, page_size=4, heads=2, dim=8):
    block = DraftBlock.__new__(DraftBlock)
    block.k_cache, block.v_cache = torch.zeros(pages, page_size, heads, dim), torch.zeros(pages, page_size, heads, dim)
    return block


def _drafted(sequences=3, tokens=5, heads=2, dim=8):
    return (torch.randn((sequences, tokens, heads, dim), generator=torch.Generator().manual_seed(i)) for i in (1, 2))


TABLE = torch.tensor([[3, 1], [0, 2], [7, 5]], dtype=torch.int32)


@pytest.mark.parametrize("accepted", [[[0], [], [1, 3, 4]], [[], [], []], [[0, 1], [2], [0]]])
def test_accepted_tokens_follow_the_committed_ones(accepted):
    block, (keys, values), lengths = _block(), _drafted(), torch.tensor([3, 8, 0], dtype=torch.int32)
    if accepted[1]:
        lengths[1] = 7
    longer = block.accept(keys, values, accepted, TABLE, lengths)
    assert longer.dtype == torch.int32 and longer.tolist() == [n + len(a) for n, a in zip(lengths.tolist(), accepted)]
    k, v = torch.zeros_like(block.k_cache), torch.zeros_like(block.v_cache)
    for i, tokens in enumerate(accepted):
        for j, t in enumerate(tokens):
            at = int(lengths[i]) + j
            k[TABLE[i, at // 4], at % 4], v[TABLE[i, at // 4], at % 4] = keys[i, t], values[i, t]
    assert torch.equal(block.k_cache, k) and torch.equal(block.v_cache, v)


@pytest.mark.parametrize("what", ["past the table", "no table", "a page that does not exist", "a negative page", "a negative length", "no such token", "too few lists"])
def test_what_has_no_place_is_refused_and_nothing_is_written(what):
    block, (keys, values), lengths, table, accepted = _block(), _drafted(), torch.tensor([3, 7, 0], dtype=torch.int32), TABLE.clone(), [[0, 1], [2], [0]]
    if what == "past the table":
        lengths[1] = 8
    elif what == "no table":
        table = table[:, :0]
    elif what == "a page that does not exist":
        table[0, 1] = 8
    elif what == "a negative page":
        table[0, 1] = -1
    elif what == "a negative length":
        lengths[2] = -1
    elif what == "no such token":
        accepted[2] = [5]
    else:
        accepted.pop()
    with pytest.raises(ValueError):
        block.accept(keys, values, accepted, table, lengths)
    assert not block.k_cache.any() and not block.v_cache.any()
