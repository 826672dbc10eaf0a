"""The 8-bit cache, attention over it, the choice among drafted tokens and the writing of the accepted ones, as they follow one another in a step
(fp6_marlin_b200.draft_step), against the same step in elementary operations.

Bound of a step's result: that of test_gpu_draft_step.py, 2e-2: both read the same 8-bit cache, so it adds nothing.
"""
import subprocess
import sys

import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200.draft_step import DraftBlock, make_inputs, plain_step
from test_gpu_verify_drafts import rule

pytestmark = pytest.mark.gpu

VOCAB = 1000


def _block(heads, kv_heads, tokens, sequences=3):
    return DraftBlock(hidden=heads * 128, inter=2816, heads=heads, kv_heads=kv_heads, sequences=sequences, tokens=tokens, pages=128, quant_cols=128, fp8_cache=True, vocab=VOCAB)


def _drafts(block, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (block.sequences, block.tokens)
    return torch.randint(VOCAB, shape, generator=gen, device="cuda"), torch.rand(shape, generator=gen, device="cuda")


@pytest.mark.parametrize("heads,kv_heads,tokens,cached", [(8, 8, 4, 100), (16, 2, 9, 300), (8, 8, 1, 50), (16, 4, 6, 200)])
def test_steps(heads, kv_heads, tokens, cached):
    """Two steps: the second sees what the first has accepted, in 8 bits."""
    block = _block(heads, kv_heads, tokens)
    x, page_table, lengths, tree = make_inputs(block, cached)
    drafted, uniforms = _drafts(block, 1)
    for _ in range(2):
        result, keys, values = block.step(x, page_table, lengths, tree)
        expect = plain_step(block, x, page_table, lengths, tree)
        assert float((result.float() - expect).norm() / expect.norm()) <= 2e-2
        accepted, counts, next_tokens = block.choose(result, drafted, tree, uniforms)
        target = torch.softmax(block.logits.float(), 1).view(block.sequences, tokens, VOCAB)
        for got, want in zip((accepted, counts, next_tokens), rule(target.cpu(), drafted.cpu(), tree.cpu(), uniforms.cpu())):
            assert torch.equal(got.cpu(), want.to(got.dtype))
        before = lengths.clone()
        block.commit(keys, values, accepted, counts, page_table, lengths)
        assert torch.equal(lengths, before + counts)
        # the accepted tokens' keys and values stand in the cache, within half a step of E4M3
        k_cache, v_cache = block.cached_values()
        for i in range(block.sequences):
            for j in range(int(counts[i])):
                at, token = int(before[i]) + j, int(accepted[i, j])
                page, slot = int(page_table[i, at // 16]), at % 16
                for cache, new in ((k_cache, keys), (v_cache, values)):
                    row = new[i, token].float()
                    assert ((cache[page, slot] - row).abs() <= torch.maximum(row.abs() * 2.0 ** -4, row.abs().amax(1, keepdim=True) * 2.0 ** -17)).all()
    assert fm.device_status() == 0
    with pytest.raises(ValueError):                                # of a 16-bit cache
        block.accept(keys, values, [[0]] * block.sequences, page_table, lengths)


def test_a_step_in_a_graph():
    """All of a step, with the cache and the lengths that it changes, captured once and replayed: the same as eager steps."""
    def run(captured):
        block = _block(16, 2, 5)
        x, page_table, lengths, tree = make_inputs(block, 150)
        table = torch.cat([page_table, torch.arange(100, 106, dtype=torch.int32, device="cuda").view(3, 2)], 1)
        lengths.clamp_(max=150)
        drafted, uniforms = _drafts(block, 2)
        seen = []

        def step():
            result, keys, values = block.step(x, table, lengths, tree)
            accepted, counts, next_tokens = block.choose(result, drafted, tree, uniforms)
            block.commit(keys, values, accepted, counts, table, lengths)
            drafted[:, 0] = next_tokens

        stream = torch.cuda.Stream()
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                step()
        previous = fm.set_ordered_sums(True)
        try:
            for _ in range(4):
                if captured:
                    graph.replay()
                else:
                    with torch.cuda.stream(stream):
                        step()
                torch.cuda.synchronize()
                seen.append([t.clone() for t in (block.accepted, block.counts, block.next_tokens, lengths, *(c.view(torch.uint8) for c in block.fp8))])
        finally:
            fm.set_ordered_sums(previous)
        return seen

    for eager, replayed in zip(run(False), run(True)):
        assert all(torch.equal(a, b) for a, b in zip(eager, replayed))
    assert fm.device_status() == 0


def test_command():
    out = subprocess.run([sys.executable, "-m", "fp6_marlin_b200.draft_step", "--sequences", "2", "--tokens", "4", "--cached", "100", "--fp8-cache"], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and "accepted tokens:" in out.stdout, out.stderr
