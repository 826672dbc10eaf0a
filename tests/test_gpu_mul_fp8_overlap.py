"""mul_fp8 with launch overlap: B is read, and counted by the barriers, before the kernel in front - which writes A and its scales - has finished.
Sums are added in one order, so the results are those without overlap bit for bit."""
import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200 import _lib
from test_gpu_mul_fp8 import SIZES, _check, _operands

pytestmark = pytest.mark.gpu

# fewer blocks of K than stages, one block, ranges over several tiles, an odd block at the end
FEW_BLOCKS = [(7, 128, 40000), (20, 16, 20000), (64, 640, 9000), (100, 128, 30000), (128, 656, 5000), (140, 384, 20000), (300, 128, 8192), (300, 400, 9000),
              (520, 640, 6000), (1030, 272, 4104), (2300, 768, 1032)]


@pytest.fixture
def overlap():
    previous = fm.set_launch_overlap(False)
    yield
    fm.set_launch_overlap(previous)


def _chain(xs, b, sb, n, dtype, repeats):
    """Rows to E4M3, product, the next rows into the same tensors, product, ..."""
    m, k = xs[0].shape
    a, sa = torch.zeros((m, k), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((m, sb.shape[1]), device="cuda")
    outs = [torch.full((m, n), float("nan"), dtype=dtype, device="cuda") for _ in range(repeats)]
    torch.cuda.synchronize()
    for i, c in enumerate(outs):
        fm.quantize_fp8(xs[i % len(xs)], a, sa)
        fm.mul_fp8(a, b, c, sa, sb)
    torch.cuda.synchronize()
    return outs, a, sa


@pytest.mark.parametrize("m,k,n", SIZES + FEW_BLOCKS)
def test_behind_the_kernel_that_writes_the_rows(m, k, n, overlap):
    dtype = torch.bfloat16 if m % 2 else torch.float16
    _, b, _, sb = _operands(1, k, n)
    xs = [torch.randn((m, k), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").to(dtype) for i in range(3)]
    expect, _, _ = _chain(xs, b, sb, n, dtype, 3)
    fm.set_launch_overlap(True)
    got, a, sa = _chain(xs, b, sb, n, dtype, 7)
    for i, c in enumerate(got):
        assert torch.equal(c, expect[i % 3])
    _check(got[-1], a, b, sa, sb)
    assert fm.device_status() == 0


def test_kernels_for_few_and_many_rows_in_turn(overlap):
    """On one stream and one scratch, each behind the other."""
    _, b, _, sb = _operands(1, 2048, 4096)
    sets = []
    for m in (3, 131, 40, 300, 1, 64, 65):
        a, _, sa, _ = _operands(m, 2048, 8)
        sets.append((a, sa, torch.empty((m, 4096), dtype=torch.float16, device="cuda")))
    expect = []
    for on in (False, True):
        fm.set_launch_overlap(on)
        for _ in range(6):
            for a, sa, c in sets:
                c.fill_(float("nan"))
                fm.mul_fp8(a, b, c, sa, sb)
        torch.cuda.synchronize()
        expect.append([c.clone() for _, _, c in sets])
    assert all(torch.equal(x, y) for x, y in zip(*expect))
    for c, (a, sa, _) in zip(expect[1], sets):
        _check(c, a, b, sa, sb)
    assert fm.device_status() == 0


@pytest.mark.parametrize("m", [16, 131, 300])
def test_a_long_kernel_in_front(m, overlap):
    """2.5 s, more than the bound of the waits: none of them has started."""
    a, b, sa, sb = _operands(m, 1024, 1024)
    want, got = (torch.zeros((m, 1024), dtype=torch.float16, device="cuda") for _ in range(2))
    fm.mul_fp8(a, b, want, sa, sb)
    torch.cuda.synchronize()
    fm.set_launch_overlap(True)
    assert _lib.lib.fp6m_debug_busy_kernel(2500, 0, torch.cuda.current_stream().cuda_stream) == _lib.OK
    fm.mul_fp8(a, b, got, sa, sb)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and fm.device_status() == 0
