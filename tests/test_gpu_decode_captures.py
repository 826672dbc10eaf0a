"""The operators of decode_ops whose first calls are captured, and two graphs of one stream, which share its scratch."""
import subprocess
import sys

import pytest
import torch

import fp6_marlin_b200 as fm
from conftest import ROOT

pytestmark = pytest.mark.gpu


def _work(tokens, vocab, seed):
    """A step of one sequence over 1500 committed tokens: buffers, and the calls that fill them in order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda").half()                       # noqa: E731
    cache, table = fm.make_cache_fp8(60, 32, 2, 128), torch.randperm(60, generator=gen, device="cuda").int()[None]
    old, lengths, start = [randn(1, 1500, 2, 128) for _ in range(2)], torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 1500, dtype=torch.int32, device="cuda")
    q, k, v = randn(1, tokens, 8, 128), randn(1, tokens, 2, 128), randn(1, tokens, 2, 128)
    tree = fm.tree_masks(torch.arange(tokens)[None] - 1).cuda()
    target = torch.softmax(2 * torch.randn((1, tokens, vocab), generator=gen, device="cuda"), 2)
    drafted, uniforms = torch.randint(vocab, (1, tokens), generator=gen, device="cuda"), torch.rand((1, tokens), generator=gen, device="cuda")
    target[0, 0, drafted[0, min(1, tokens - 1)]] = 1.0                                                   # (a token that is accepted)
    outs = [torch.zeros_like(q), torch.zeros((1, tokens), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda"),
            *(torch.zeros((1, 1500 + tokens, 2, 128), dtype=torch.half, device="cuda") for _ in range(2))]

    def call():
        fm.write_cache_fp8(*old, *cache, table, lengths)
        fm.tree_attention_fp8(q, k, v, *cache, table, start, tree, outs[0])
        fm.verify_drafts(target, drafted, tree, uniforms, *outs[1:4])
        fm.write_cache_fp8(k, v, *cache, table, start, tokens=outs[1], counts=outs[2])
        fm.read_cache_fp8(*cache, table, start + outs[2], *outs[4:])

    return call, outs


def first_calls_in_a_capture():
    works = [_work(3, 140000, 1), _work(20, 3000, 2)]
    stream, graphs = torch.cuda.Stream(), [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, (call, _) in zip(graphs, works):
        with torch.cuda.graph(graph, stream=stream):
            call()
            call()
    seen = {}
    for which in (1, 1, 0, 1, 0, 0):
        for x in works[which][1]:
            x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[which].replay()
        torch.cuda.synchronize()
        now = [x.clone() for x in works[which][1]]
        assert all(torch.equal(x, y) for x, y in zip(now, seen.setdefault(which, now)))
    for which, (call, outs) in enumerate(works):
        for x in outs:
            x.zero_()
        call()                                                                                           # on another stream, with scratch of its own
        assert all(torch.equal(x, y) for x, y in zip(outs, seen[which])) and int(outs[2]) >= 2 and float(outs[0].abs().sum()) > 0
    assert fm.device_status() == 0


def test_first_calls_of_a_process_in_a_capture():
    program = "import sys; sys.path[:0] = ['.', 'tests']; import test_gpu_decode_captures as t; t.first_calls_in_a_capture(); print('ok')"
    run = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout[-2000:] + run.stderr[-2000:]
