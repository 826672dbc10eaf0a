"""rms_norm and quantize_fp8 against the formulas in 64 bits.

Bounds: a result rounded once to a type with p significant bits is off by at most 2^-p of itself (fp16 p = 11, bf16 8, E4M3 4) or half the
type's smallest step; the fp32 arithmetic before it (a sum of N squares in a tree whose leaves add at most 64 values, a reciprocal root,
three products) stays below 80 * 2^-24 < 2^-17 of the value.
"""
import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu

BITS = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}
ARITHMETIC = 2.0 ** -17


def _rows(m, n, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 7 * m + n)
    return (torch.randn((m, n), generator=gen, device="cuda") * scale).to(dtype)


def _norm64(x, w, eps, r=None):
    h = x.double() if r is None else x.double() + r.double()
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()


def _close(got, expect, dtype):
    rel, step = BITS[dtype]
    bound = (rel + ARITHMETIC) * expect.abs() + step
    assert ((got.double() - expect).abs() <= bound).all(), float(((got.double() - expect).abs() / bound).max())


def _scales64(y):
    m, n = y.shape
    padded = torch.nn.functional.pad(y.abs(), (0, -n % 128)).view(m, -1, 128)
    return padded.amax(2).clamp(min=1e-30) / 448


def _check_fp8(q, s, y):
    s64 = _scales64(y)
    assert ((s.double() - s64).abs() <= ARITHMETIC * s64).all()
    ratio = y / s64.repeat_interleave(128, 1)[:, :y.shape[1]]
    bound = (ratio.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) * (1 + 2.0 ** -10) + 448 * ARITHMETIC
    assert ((q.double() - ratio).abs() <= bound).all()


SIZES = [(1, 8), (1, 4096), (3, 136), (5, 120), (2, 1024), (37, 8192), (7, 4104), (300, 512), (3, 16384), (2, 28672), (1, 65544), (1001, 2056)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(m, n, dtype, residual):
    x, w = _rows(m, n, dtype), _rows(1, n, dtype, 1)[0]
    r = _rows(m, n, dtype, 2, 3.0) if residual else None
    h, y64 = _norm64(x, w, 1e-5, r)
    y, total = torch.full_like(x, 7), torch.full_like(x, 7) if residual else None
    fm.rms_norm(x, w, y, 1e-5, residual=r, residual_out=total)
    _close(y, y64, dtype)
    if residual:
        assert torch.equal(total, (x.float() + r.float()).to(dtype))
    q, s = torch.empty((m, n), dtype=torch.float8_e4m3fn, device="cuda"), torch.full((m, -(-n // 128)), 7.0, device="cuda")
    fm.rms_norm(x, w, q, 1e-5, scales=s, residual=r)               # the residual in place
    _check_fp8(q, s, y64)
    if residual:
        assert torch.equal(r, total)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n", SIZES)
def test_quantize(m, n, dtype):
    x = _rows(m, n, dtype, 3, 5.0)
    x[0, : n // 2] = 0                                             # groups of zeros
    q, s = torch.empty((m, n), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((m, -(-n // 128)), device="cuda")
    fm.quantize_fp8(x, q, s)
    _check_fp8(q, s, x.double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_extremes(dtype):
    """Rows of zeros, of the type's largest values (whose sum overflows the stored residual, not the norm), and with NaN."""
    n, top = 512, torch.finfo(dtype).max
    x = torch.zeros((4, n), dtype=dtype, device="cuda")
    x[1] = top
    x[2, 5] = float("nan")
    x[3] = 1
    w = torch.ones(n, dtype=dtype, device="cuda")
    r = x.clone()
    y, total = torch.empty_like(x), torch.empty_like(x)
    fm.rms_norm(x, w, y, 1e-6, residual=r, residual_out=total)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and total[1].isinf().all() and y[2].isnan().all()
    assert (y[3].float() - 1).abs().max() <= BITS[dtype][0] + ARITHMETIC
    if dtype == torch.float16:
        assert (y[1].float() - 1).abs().max() <= BITS[dtype][0] + ARITHMETIC
    q, s = torch.empty((4, n), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((4, 4), device="cuda")
    fm.quantize_fp8(x, q, s)
    assert (q[0].float() == 0).all() and (s[0] > 0).all() and (q[1].float() == 448).all()
    assert s[2, 0].isnan() and q[2, 5].float().isnan() and (s[2, 1:] > 0).all() and (q[2, 128:].float() == 0).all()


def test_runs_on_the_current_stream_and_in_a_graph():
    x, w = _rows(33, 4096, torch.float16), torch.ones(4096, dtype=torch.float16, device="cuda")
    expect, y = torch.empty_like(x), torch.zeros_like(x)
    fm.rms_norm(x, w, expect)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            fm.rms_norm(x, w, y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, expect)


def test_no_rows_and_refusals():
    x, w = _rows(4, 256, torch.float16), torch.ones(256, dtype=torch.float16, device="cuda")
    q, s = torch.empty((4, 256), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((4, 2), device="cuda")
    fm.rms_norm(x[:0], w, torch.empty_like(x[:0]))
    fm.quantize_fp8(x[:0], q[:0], s[:0])
    y = torch.empty_like(x)
    for bad in (lambda: fm.rms_norm(x.float(), w, y), lambda: fm.rms_norm(x, w.float(), y), lambda: fm.rms_norm(x, w[:128], y),
                lambda: fm.rms_norm(x, w, y[:2]), lambda: fm.rms_norm(x, w, q), lambda: fm.rms_norm(x, w, y, scales=s),
                lambda: fm.rms_norm(x, w, q, scales=s[:, :1]), lambda: fm.rms_norm(x.t().contiguous().t(), w, y),
                lambda: fm.rms_norm(x, w, y, residual_out=y), lambda: fm.rms_norm(x, w, y, residual=x[:2]),
                lambda: fm.rms_norm(x[:, :252].contiguous(), w[:252], y[:, :252].contiguous()), lambda: fm.rms_norm(x.cpu(), w, y),
                lambda: fm.rms_norm(x, w.cpu(), y), lambda: fm.quantize_fp8(x, q, None), lambda: fm.quantize_fp8(x, y, s),
                lambda: fm.quantize_fp8(x, q, s.half()), lambda: fm.rms_norm(x.flatten()[4:4 + 512].view(2, 256), w, y[:2])):
        with pytest.raises(RuntimeError):
            bad()


def test_rows_as_long_as_an_int_can_say():
    """Two rows of 2^31 - 8 values: the scales and values of the second lie where they belong."""
    n = (1 << 31) - 8
    x = torch.full((2, n), 1.0, dtype=torch.bfloat16, device="cuda")
    top = torch.full((2, -(-n // 128)), 1.0, device="cuda")
    spots = [1, 100, 128, n // 2 - 50, n - 200, n - 120, n - 1]      # the last group has 120 values
    for i, at in enumerate(spots):
        x[1, at] = -2.0 - i
        top[1, at // 128] = 2.0 + i                                  # (a later spot is larger)
    q, s = torch.empty((2, n), dtype=torch.float8_e4m3fn, device="cuda"), torch.full_like(top, 7.0)
    fm.quantize_fp8(x, q, s)
    assert ((s.double() * 448 - top).abs() <= ARITHMETIC * top).all()
    for first in (0, 128, n // 2 // 128 * 128, n - 248, n - 120):
        _check_fp8(q[:, first:first + 120], s[:, first // 128][:, None], x[:, first:first + 120].double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_are_divided_by_the_scale_that_is_stored(dtype):
    """Bit for bit, also where the quotient lies on the boundary between two E4M3 values: few distinct values, so that many do."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = (torch.randint(-255, 256, (301, 2056), generator=gen, device="cuda") * torch.exp2(torch.randint(-6, 3, (301, 1), generator=gen, device="cuda"))).to(dtype)
    q, s = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((301, 17), device="cuda")
    fm.quantize_fp8(x, q, s)
    top = torch.nn.functional.pad(x.float().abs(), (0, 120)).view(301, 17, 128).amax(2).clamp(min=1e-30).cpu()
    assert torch.equal(s.cpu(), top * torch.tensor(1.0 / 448.0))     # (one product in fp32)
    expect = (x.float().cpu() / s.cpu().repeat_interleave(128, 1)[:, :2056]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(q.cpu().view(torch.uint8), expect.view(torch.uint8))


def test_division_by_infinite_and_by_small_scales():
    x = torch.zeros((6, 128), dtype=torch.bfloat16, device="cuda")
    x[:, ::3] = 1.0
    x[0, 5], x[1, 7] = float("inf"), float("-inf")                   # finite values by infinity are 0
    x[2] *= 1e-30
    x[3], x[3, 9] = 1e-39, 1e-31                                     # below the least scale
    x[4], x[4, 1] = torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).min
    x[5] *= torch.linspace(1e-38, 1e-30, 128, device="cuda")
    q, s = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((6, 1), device="cuda")
    fm.quantize_fp8(x, q, s)
    top = x.float().abs().amax(1, keepdim=True).clamp(min=1e-30).cpu()
    assert torch.equal(s.cpu(), top * torch.tensor(1.0 / 448.0))     # (one product in fp32)
    expect = (x.float().cpu() / s.cpu()).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    assert torch.equal(q.cpu().float().nan_to_num(nan=1000.0), expect.nan_to_num(nan=1000.0)) and int(q.float().isnan().sum()) == 2


def test_misaligned_tensors_are_named():
    x, w = _rows(2, 256, torch.float16), torch.ones(264, dtype=torch.float16, device="cuda")
    q, s = torch.empty(520, dtype=torch.uint8, device="cuda")[8:].view(torch.float8_e4m3fn).view(2, 256), torch.empty((2, 2), device="cuda")
    b, c = torch.empty((8, 256), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((2, 8), dtype=torch.float16, device="cuda")
    for call in (lambda: fm.rms_norm(x, w[4:260], torch.empty_like(x)), lambda: fm.rms_norm(x, w[:256], q, scales=s), lambda: fm.quantize_fp8(x, q, s),
                 lambda: fm.mul_fp8(q, b, c, s, s[:1])):
        with pytest.raises(RuntimeError, match="16-byte boundaries"):
            call()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(37, 8192), (301, 2056), (5, 30000)])
def test_quantised_rows_are_those_of_torch_operations(m, n, dtype):
    """On the GPU, where torch divides by a number as a product with its reciprocal and by a tensor with one rounding."""
    x = _rows(m, n, dtype, 9, 3.0)
    q, s = torch.empty((m, n), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((m, -(-n // 128)), device="cuda")
    fm.quantize_fp8(x, q, s)
    scales = torch.nn.functional.pad(x.float(), (0, -n % 128)).view(m, -1, 128).abs().amax(2).clamp(min=1e-30) / 448
    expect = (x.float() / scales.repeat_interleave(128, 1)[:, :n]).to(torch.float8_e4m3fn)
    assert torch.equal(s, scales) and torch.equal(q.view(torch.uint8), expect.view(torch.uint8))
