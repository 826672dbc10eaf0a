"""mul_fp8 against sums in 64 bits.

Bounds: one rounding to a type with p significant bits (fp16 11, bf16 8), 2^-p of the result at most, and K additions in fp32, each
off by at most 2^-23 of a partial sum (rounded or truncated): K * 2^-23 of the sum of magnitudes.  In the mean over a matrix the
rounding alone is below 2^-p / sqrt(3), and the additions do not reach the rest.
"""
import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu

BITS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _operands(m, k, n, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + m + 3 * k + 7 * n)
    a = (torch.randn((m, k), generator=gen, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    b = (torch.randn((n, k), generator=gen, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    kb, nb = -(-k // 128), -(-n // 128)
    # scales of very different sizes, so that one in the wrong place shows
    sa = torch.exp2(torch.rand((m, kb), generator=gen, device="cuda") * 8 - 12)
    sb = torch.exp2(torch.rand((nb, kb), generator=gen, device="cuda") * 8 - 12)
    return a, b, sa, sb


def _exact(a, b, sa, sb):
    (m, k), n = a.shape, b.shape[0]
    a64 = a.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    b64 = b.double() * sb.double().repeat_interleave(128, 1)[:, :k].repeat_interleave(128, 0)[:n]
    return a64 @ b64.T, a64.abs() @ b64.abs().T


def _check(c, a, b, sa, sb):
    expect, size = _exact(a, b, sa, sb)
    k = a.shape[1]
    err = (c.double() - expect).abs()
    bound = BITS[c.dtype] * expect.abs() + k * 2.0 ** -23 * size + 2.0 ** -25
    assert (err <= bound).all(), float((err / bound).max())
    assert float(err.norm() / expect.norm()) <= BITS[c.dtype] / 3 ** 0.5


SIZES = [(1, 16, 8), (1, 4096, 4096), (2, 144, 136), (3, 128, 128), (5, 4096, 1024), (8, 2048, 264), (9, 11008, 512), (16, 8192, 2048), (17, 1040, 4104),
         (31, 512, 10240), (32, 4096, 12288), (33, 4112, 640), (48, 1024, 520), (64, 8192, 4096), (65, 256, 1032), (100, 11008, 4096), (127, 400, 2056),
         (128, 4096, 4096), (129, 4096, 4096), (131, 11008, 4096), (200, 1536, 8), (255, 384, 5000), (256, 2048, 2048), (257, 8192, 1280), (513, 4096, 4104),
         (777, 4096, 11008), (1024, 128, 4096), (1500, 4112, 2824), (2048, 2048, 8192), (4099, 512, 776)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_product(m, k, n, dtype):
    a, b, sa, sb = _operands(m, k, n)
    c = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    for _ in range(2):                                             # a second run finds the scratch as the first left it
        c.fill_(float("nan"))
        fm.mul_fp8(a, b, c, sa, sb)
        _check(c, a, b, sa, sb)
    again = torch.empty_like(c)
    fm.mul_fp8(a, b, again, sa, sb)
    assert torch.equal(c, again)                                   # sums are added in one order


@pytest.mark.parametrize("m", [1, 7, 20, 40, 90, 150, 300])
def test_every_block_and_row_counts_once(m):
    """Ones everywhere, scales that are powers of two: the result is exact, so a block left out or taken twice shows."""
    k, n = 2064, 1288
    a, b = torch.ones((m, k), device="cuda").to(torch.float8_e4m3fn), torch.ones((n, k), device="cuda").to(torch.float8_e4m3fn)
    kb, nb = -(-k // 128), -(-n // 128)
    sa = torch.exp2(-(torch.arange(m, device="cuda") % 5).float())[:, None].expand(m, kb).contiguous()
    sb = torch.exp2(-(torch.arange(nb, device="cuda") % 3).float())[:, None].expand(nb, kb).contiguous()
    c = torch.empty((m, n), dtype=torch.float16, device="cuda")
    fm.mul_fp8(a, b, c, sa, sb)
    expect = k * sa[:, :1] * sb[:, 0].repeat_interleave(128)[:n]
    assert torch.equal(c.float(), expect)


@pytest.mark.parametrize("m", [1, 24, 100, 300])
def test_nan_and_large_values_stay_in_their_places(m):
    a, b, sa, sb = _operands(m, 512, 256)
    sb[:] = 2.0 ** -12
    sa[:] = 2.0 ** -12
    a[0, 3] = float("nan")
    sa[m - 1, 1] = 2.0 ** 120 if m > 1 else sa[m - 1, 1]
    c = torch.empty((m, 256), dtype=torch.bfloat16, device="cuda")
    fm.mul_fp8(a, b, c, sa, sb)
    assert c[0].isnan().all()
    if m > 2:
        assert c[1:m - 1].isfinite().all()
        _check(c[1:m - 1], a[1:m - 1], b, sa[1:m - 1], sb)
        assert c[m - 1].abs().max() > 2.0 ** 100


def test_streams_and_graph():
    """Two streams at once (a scratch each), and a captured call that is replayed."""
    sets = [_operands(24, 8192, 1024, seed) for seed in (1, 2)]
    outs = [torch.empty((24, 1024), dtype=torch.float16, device="cuda") for _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, c, st in zip(sets, outs, streams):
            with torch.cuda.stream(st):
                fm.mul_fp8(x[0], x[1], c, x[2], x[3])
    torch.cuda.synchronize()
    for x, c in zip(sets, outs):
        _check(c, *x)
    graph, c = torch.cuda.CUDAGraph(), torch.empty_like(outs[0])
    a, b, sa, sb = sets[0]
    with torch.cuda.graph(graph, stream=streams[0]):
        fm.mul_fp8(a, b, c, sa, sb)
    for _ in range(3):
        c.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, outs[0]) and fm.device_status() == 0


def test_weights_of_make_fp8_weight():
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn((520, 1040), generator=gen, device="cuda") * 0.02
    q, s = fm.make_fp8_weight(w)
    x = torch.randn((9, 1040), generator=gen, device="cuda").half()
    xq, xs = torch.empty((9, 1040), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((9, 9), device="cuda")
    fm.quantize_fp8(x, xq, xs)
    c = torch.empty((9, 520), dtype=torch.float16, device="cuda")
    fm.mul_fp8(xq, q, c, xs, s)
    _check(c, xq, q, xs, s)
    expect = x.double() @ w.double().T
    # each factor is off by at most 2^-4 of itself, uniformly 2^-4 / sqrt(3) or less in the mean
    assert float((c.double() - expect).norm() / expect.norm()) <= 2 ** 0.5 * 2.0 ** -4 / 3 ** 0.5


def test_no_terms_no_rows_and_refusals():
    a, b, sa, sb = _operands(4, 256, 128)
    c = torch.full((4, 128), 7.0, dtype=torch.float16, device="cuda")
    fm.mul_fp8(a[:, :0].contiguous(), b[:, :0].contiguous(), c, sa[:, :0].contiguous(), sb[:, :0].contiguous())
    assert (c == 0).all()
    fm.mul_fp8(a[:0], b, c[:0], sa[:0], sb)
    fm.mul_fp8(a, b[:0], c[:, :0], sa, sb[:0])
    odd = torch.zeros(4 * 256 + 8, dtype=torch.uint8, device="cuda")[8:].view(torch.float8_e4m3fn).view(4, 256)
    for bad in (lambda: fm.mul_fp8(a.float(), b, c, sa, sb), lambda: fm.mul_fp8(a, b, c.float(), sa, sb), lambda: fm.mul_fp8(a, b, c[:, :64], sa, sb),
                lambda: fm.mul_fp8(a[:, :128], b[:, :128], c, sa[:, :1].contiguous(), sb[:, :1].contiguous()), lambda: fm.mul_fp8(a, b, c, sa.half(), sb),
                lambda: fm.mul_fp8(a, b, c, sa[:, :1], sb), lambda: fm.mul_fp8(a, b, c, sa, sb.repeat(2, 1)), lambda: fm.mul_fp8(a.cpu(), b, c, sa, sb),
                lambda: fm.mul_fp8(a, b.cpu(), c, sa, sb), lambda: fm.mul_fp8(odd, b, c, sa, sb), lambda: fm.mul_fp8(a, b[:, :128], c, sa, sb),
                lambda: fm.mul_fp8(a[:, :8].contiguous(), b[:, :8].contiguous(), c, sa[:, :1].contiguous(), sb[:, :1].contiguous()),
                lambda: fm.mul_fp8(a, b[:100].contiguous(), c[:, :100].contiguous(), sa, sb)):
        with pytest.raises(RuntimeError):
            bad()
