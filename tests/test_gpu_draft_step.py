"""A decoder block's step over drafted trees (fp6_marlin_b200.draft_step) against the same step in elementary operations.

Bound: both round rows to E4M3; upstream results differ by fp16 roundings (a few times 2^-11), so that about one value in 2^-3 / 2^-10 = 128
falls on the other side of a rounding boundary and then differs by up to 2^-3 of itself: sqrt(1/128) * 2^-3 = 1.1e-2 of the rows of either
product, and the block's result carries part of it: 2e-2.
"""
import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200.draft_step import DraftBlock, make_inputs, plain_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,tokens,cached", [(8, 8, 4, 100), (16, 2, 9, 300)])
def test_step(heads, kv_heads, tokens, cached):
    block = DraftBlock(hidden=heads * 128, inter=2816, heads=heads, kv_heads=kv_heads, sequences=3, tokens=tokens, pages=128, quant_cols=128)
    x, page_table, lengths, tree = make_inputs(block, cached)
    result, keys, values = block.step(x, page_table, lengths, tree)
    expect = plain_step(block, x, page_table, lengths, tree)
    assert float((result.float() - expect).norm() / expect.norm()) <= 2e-2
    # accepted tokens become committed ones: the next step sees them in the cache as it saw them among the drafted
    accepted = [[0], [], [0, 1] if int(tree[2, 1]) & 1 else [0]]
    longer = block.accept(keys, values, accepted, page_table, lengths)
    assert longer.tolist() == [n + len(a) for n, a in zip(lengths.tolist(), accepted)]
    again, _, _ = block.step(x, page_table, longer, tree)
    expect = plain_step(block, x, page_table, longer, tree)
    assert float((again.float() - expect).norm() / expect.norm()) <= 2e-2
    assert fm.device_status() == 0
