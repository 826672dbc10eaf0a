"""What a wait that ran out may leave in an operator's scratch does not reach later calls: device_status, which reports it, makes the scratch as it was before the first call.

No wait runs out here: the words that a late CTA would leave, and the status, are stored from the host.
"""
import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200 import _lib, api, block_ops
from test_gpu_tree_attention_fp8 import NAMES, inputs, run

pytestmark = pytest.mark.gpu


def _leave_words(stream, status):
    for buffer in block_ops._scratch["tree_attention_fp8", 0, stream.cuda_stream]:
        buffer.fill_(0x3c)                                           # (as floats: 0.0115)
    api._status[0].fill_(status)
    torch.cuda.synchronize()


# (a bad page may be reported in the same word after the wait)
@pytest.mark.parametrize("status", [_lib.ERR_TIMEOUT, _lib.ERR_BAD_ARG])
@pytest.mark.parametrize("t,h,g,d", [(1, 4, 1, 128), (3, 4, 1, 64), (9, 2, 1, 128), (32, 1, 1, 64), (40, 8, 2, 64)])
def test_calls_after_a_status(t, h, g, d, status):
    """One sequence and few heads of keys: every multiprocessor leaves a part of the same rows, and the parts are joined."""
    x = inputs(1, t, h, g, d, [24690], 16)
    expect = run(x)
    assert fm.device_status() == 0
    _leave_words(torch.cuda.current_stream(), status)
    assert fm.device_status() == status and fm.device_status() == 0
    for _ in range(3):
        assert torch.equal(run(x), expect)
    assert fm.device_status() == 0


def test_replays_after_a_status():
    """A captured call has its stream's scratch for good."""
    x = inputs(1, 2, 4, 1, 128, [24690], 16)
    expect, out = run(x), torch.zeros(x["q"].shape, dtype=x["q"].dtype, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        fm.tree_attention_fp8(*(x[n] for n in NAMES), out)
    _leave_words(stream, _lib.ERR_TIMEOUT)
    assert fm.device_status() == _lib.ERR_TIMEOUT
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, expect)
    assert fm.device_status() == 0
