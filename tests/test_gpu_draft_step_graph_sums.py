"""A captured step of DraftBlock with an 8-bit cache against eager ones, both with ordered sums: 15 rows, and 48, where the products by INT4 / FP6 weights add in an order of their own without the switch."""
import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200.draft_step import make_inputs
from test_gpu_draft_step_fp8 import _block, _drafts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [5, 16])
def test_a_captured_step_with_ordered_sums(tokens):
    def run(captured):
        block = _block(16, 2, tokens)
        x, page_table, lengths, tree = make_inputs(block, 150)
        more = 3 * (-(-4 * tokens // 16) + 1)
        free = torch.tensor(sorted(set(range(128)) - set(page_table.flatten().tolist()))[:more], dtype=torch.int32, device="cuda")
        table = torch.cat([page_table, free.view(3, -1)], 1)
        drafted, uniforms = _drafts(block, 2)
        seen, stream, graph = [], torch.cuda.Stream(), torch.cuda.CUDAGraph()

        def step():
            result, keys, values = block.step(x, table, lengths, tree)
            accepted, counts, next_tokens = block.choose(result, drafted, tree, uniforms)
            block.commit(keys, values, accepted, counts, table, lengths)
            drafted[:, 0] = next_tokens

        torch.cuda.synchronize()
        if captured:
            with torch.cuda.graph(graph, stream=stream):
                step()
        for _ in range(4):
            with torch.cuda.stream(stream):
                graph.replay() if captured else step()
            torch.cuda.synchronize()
            seen.append([t.clone() for t in (block.result, block.accepted, block.counts, block.next_tokens, lengths, *(c.view(torch.uint8) for c in block.fp8))])
        return seen

    previous = fm.set_ordered_sums(True)                           # (read when a product is launched or captured)
    try:
        for eager, replayed in zip(run(False), run(True)):
            assert all(torch.equal(a, b) for a, b in zip(eager, replayed))
    finally:
        fm.set_ordered_sums(previous)
    assert fm.device_status() == 0
