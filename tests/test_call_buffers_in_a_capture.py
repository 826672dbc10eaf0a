"""A scratch or status word that is first needed while a stream is being captured into a graph: zero from the start, and never again
because of a replay."""
import contextlib
import subprocess
import sys
import types

import pytest
import torch

import fp6_marlin_b200 as fm
from conftest import ROOT
from fp6_marlin_b200 import api, block_ops, synth

DEV, STREAM = torch.device("cuda", 63), 7


@pytest.mark.parametrize("capturing", [False, True])
def test_buffers_are_not_made_by_operations_that_are_captured(monkeypatch, capturing):
    made, zeros = [], torch.zeros
    recorder = types.SimpleNamespace(**{n: lambda *a: None for n in ("set_scratch", "set_device", "set_operator_scratch")})
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda index: types.SimpleNamespace(multi_processor_count=148))
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch, "zeros", lambda *args, device=None, **kw: made.append("in order of the stream") or zeros(*args, **kw))
    monkeypatch.setattr(api, "_zeroed_outside_a_capture", lambda nbytes, device: made.append("at once") or zeros(nbytes, dtype=torch.uint8), raising=False)
    for module in (api, block_ops):
        monkeypatch.setattr(module, "_call", recorder)
        monkeypatch.setattr(module, "_scratch", {})
    for module, name in ((api, "_scratch_need"), (api, "_status"), (block_ops, "_status"), (api, "_sm_count"), (block_ops, "_sm_count")):
        monkeypatch.setattr(module, name, {})
    monkeypatch.setattr(block_ops, "_status", api._status)
    api._device_buffers(DEV, (1, 1024, 1024, 0), STREAM)                       # status word and scratch
    api._device_buffers(DEV, (128, 8192, 8192, 256), STREAM)                   # a larger one
    first, status = block_ops._operator_buffers("mul_fp8", DEV, 1000, STREAM)
    second, _ = block_ops._operator_buffers("mul_fp8", DEV, 5000, STREAM)
    assert made == ["at once" if capturing else "in order of the stream"] * 5
    assert first.numel() == 1000 and second.numel() == 5000 and status is api._status[63] and status.dtype == torch.int32 and status.shape == (1,)


def _unused_stream():
    used = {key[-1] for key in (*api._scratch, *block_ops._scratch)}
    return next(s for s in (torch.cuda.Stream(priority=-1) for _ in range(64)) if s.cuda_stream not in used)


def _calls(kind):
    """Two calls of an operator that need scratch of different sizes: (call, output) each."""
    out = []
    for size in (1, 2):
        if kind == "mul":
            w = synth.make_layer(1024, 1024 * size, 256, 128, seed=1, keep_dequantized=False).to(torch.device("cuda", 0))
            a, c = synth.make_activations(8 * size, 1024, 2).cuda(), torch.zeros((8 * size, 1024 * size), dtype=torch.float16, device="cuda")
            ws = torch.zeros(1024 * size // 128 * 16, dtype=torch.int32, device="cuda")
            out.append((lambda a=a, w=w, c=c, ws=ws: fm.mul(a, w.B, c, w.s, ws, 256, group_size=128, layout="b200"), c))
        elif kind.startswith("mul_fp8"):
            import test_gpu_mul_fp8 as t
            x = t._operands(int(kind.split()[1]), 8192, 1024 * size)
            c = torch.zeros((x[0].shape[0], x[1].shape[0]), dtype=torch.float16, device="cuda")
            out.append((lambda x=x, c=c: fm.mul_fp8(x[0], x[1], c, x[2], x[3]), c))
        else:
            import test_gpu_tree_attention as t
            x = t._inputs(1, int(kind.split()[1]), 16, 2, 128, [5000 * size], 16)
            c = torch.zeros_like(x["q"].contiguous())
            out.append((lambda x=x, c=c: fm.tree_attention(*(x[n] for n in ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")), c), c))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["mul", "mul_fp8 9", "mul_fp8 131", "mul_fp8 300", "tree_attention 2", "tree_attention 30"])
def test_graphs_of_a_stream_without_a_call_before(kind):
    """Whichever graph is replayed first, and with calls between them."""
    calls = _calls(kind)
    expect = []
    for call, c in calls:
        call()
        expect.append(c.clone())
    junk = torch.full((256 << 20,), 255, dtype=torch.uint8, device="cuda")       # what memory that nobody zeroes may hold
    del junk
    torch.cuda.synchronize()
    stream, graphs = _unused_stream(), [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, (call, _) in zip(graphs, calls):
        with torch.cuda.graph(graph, stream=stream):
            call()
            call()
    for which in (1, 1, 0, "call", 1, 0, "call", 0):
        for _, c in calls:
            c.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i in (0, 1) if which == "call" else (which,):
                calls[i][0]() if which == "call" else graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1) if which == "call" else (which,):
            assert torch.equal(calls[i][1], expect[i])
    assert fm.device_status() == 0


def first_call_in_a_capture():
    import test_gpu_tree_attention as t
    x = t._inputs(1, 2, 4, 1, 64, [40], 16)
    good, bad = (torch.zeros_like(x["q"].contiguous()) for _ in range(2))
    call = lambda table, out: fm.tree_attention(x["q"], x["k"], x["v"], x["k_cache"], x["v_cache"], table, x["lengths"], x["tree"], out)     # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(x["page_table"], good)
    missing = x["page_table"].clone()
    missing[0, 1] = -1
    call(missing, bad)
    graph.replay()                                                              # must not clear what the call reported
    assert fm.device_status() == 4 and fm.device_status() == 0
    t._check(good, x)


@pytest.mark.gpu
def test_first_call_of_a_process_in_a_capture():
    program = "import sys; sys.path[:0] = ['.', 'tests']; import test_call_buffers_in_a_capture as t; t.first_call_in_a_capture(); print('ok')"
    run = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout[-2000:] + run.stderr[-2000:]
