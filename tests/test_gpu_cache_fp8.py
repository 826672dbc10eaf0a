"""write_cache_fp8 and read_cache_fp8 against the rule in exact arithmetic: every stored byte, every value that is read back, and all that must be left alone.

A value of 16 bits times a power of two is exact in 64 bits, so the E4M3 value nearest to it is known (ties to the even one), and no tolerance is needed.
"""
import itertools

import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu

RANGES = {torch.float16: (-15, 8), torch.bfloat16: (-40, 120)}
# the finite E4M3 values that are not negative, by their bytes 0 .. 126
VALUES = torch.tensor([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127], dtype=torch.float64)


def encoded(x):
    """x (..., D) on the CPU -> bytes of E4M3 (NaN: 127) and exponents + 127, from the definition."""
    lowest, highest = RANGES[x.dtype]
    x = x.double()
    finite = x.isfinite()
    top = torch.where(finite, x.abs(), 0).amax(-1)
    e = torch.full(top.shape, highest)
    for power in range(highest - 1, lowest - 1, -1):               # the least one that will do
        e = torch.where(top <= 448 * 2.0 ** power, power, e)
    limit = torch.where(e == highest, 240.0, 448.0)[..., None]
    y = torch.minimum(torch.where(finite, x.abs(), 0) / torch.pow(2.0, e.double())[..., None], limit)
    above = torch.searchsorted(VALUES, y.contiguous()).clamp(max=126)
    below = (above - 1).clamp(min=0)
    up, down = VALUES[above] - y, y - VALUES[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    code = torch.where(finite, code + 128 * (torch.signbit(x) & finite), 127)
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def same_bytes(got, expect):
    """Equal but for the sign of NaN and of zero."""
    plain = lambda t: torch.where((t & 127) == 127, 127, torch.where(t == 128, 0, t))          # noqa: E731
    return torch.equal(plain(got.cpu()), plain(expect))


def cache(pages, page, g, d, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    made = list(fm.make_cache_fp8(pages, page, g, d))
    for t in made:
        t.view(torch.uint8).copy_(torch.randint(0, 255, t.shape, generator=gen, device="cuda", dtype=torch.uint8) & 0x7e)      # (no NaN)
    return made


def data(b, t, g, d, dtype, seed=0):
    """Heads of all sizes, of zeros, with the type's largest and least values, infinities and NaN."""
    gen = torch.Generator().manual_seed(seed + 13 * b + t)
    x = torch.randn((b, t, g, d), generator=gen) * torch.exp2(torch.randint(-20, 14, (b, t, g, 1), generator=gen).float())
    x = x.to(dtype)
    flat, info = x.view(-1, d), torch.finfo(dtype)
    for i, values in enumerate([(0.0,), (info.max,), (info.smallest_normal,), (float("inf"), 3.0), (float("nan"), -2.0), (448.0,), (449.0,), (float("-inf"),), (info.max, float("nan")), (-0.0, 1.75)]):
        if i < flat.shape[0]:
            flat[i] = 0
            flat[i, : len(values)] = torch.tensor(values, dtype=dtype)
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,g,d,page,listed", [(1, 1, 1, 64, 1, False), (1, 1, 1, 128, 16, False), (3, 5, 8, 128, 16, True), (2, 300, 4, 64, 24, False), (5, 64, 1, 128, 7, True), (2, 33, 40, 64, 256, False),
                                                 (1, 1000, 2, 128, 16, False), (17, 3, 5, 64, 3, True)])
def test_write_and_read(b, t, g, d, page, listed, dtype):
    gen = torch.Generator().manual_seed(b + t)
    lengths = torch.randint(0, 50, (b,), generator=gen, dtype=torch.int32)
    per = -(-(50 + t) // page)
    pages = b * per + 3
    table = torch.randperm(pages, generator=gen)[: b * per].view(b, per).int()
    k, v = data(b, t, g, d, dtype, 1), data(b, t, g, d, dtype, 2)
    made = cache(pages, page, g, d)
    expect = [x.view(torch.uint8).cpu().clone() for x in made]
    tokens = counts = None
    order = [list(range(t)) for _ in range(b)]
    if listed:                                                     # some tokens, out of order, with gaps, some of them behind the count
        tokens = torch.randint(-1, t, (b, t + 2), generator=gen, dtype=torch.int32)
        counts = torch.randint(0, t + 4, (b,), generator=gen, dtype=torch.int32)
        counts[0] = t + 2
        lengths[-1] = 0
        order = [row[: max(0, n)] for row, n in zip(tokens.tolist(), counts.tolist())]
    per_tokens = per * page
    for i, row in enumerate(order):
        for j, token in enumerate(row):
            at = int(lengths[i]) + j
            if token < 0 or at >= per_tokens:
                continue
            page_of, slot = int(table[i, at // page]), at % page
            for n, x in enumerate((k, v)):
                code, power = encoded(x[i, token])
                expect[n][page_of, slot], expect[2 + n][page_of, slot] = code, power
    fits = not any(token >= 0 and int(lengths[i]) + j >= per_tokens for i, row in enumerate(order) for j, token in enumerate(row))
    on = lambda x: None if x is None else x.cuda()                  # noqa: E731
    args = [table.cuda(), lengths.cuda()]
    fm.write_cache_fp8(k.cuda(), v.cuda(), *made, *args, tokens=on(tokens), counts=on(counts))
    assert fm.device_status() == (0 if fits else 4)
    for got, want in zip(made, expect):
        assert same_bytes(got.view(torch.uint8), want) if got.dtype == torch.float8_e4m3fn else torch.equal(got.cpu(), want)

    # back: all rows, then a stretch from somewhere (before the first token, too)
    longer = torch.tensor([min(n + len(row), per_tokens) for n, row in zip(lengths.tolist(), order)], dtype=torch.int32)
    for rows, starts in ((per_tokens + 2, None), (20, torch.randint(-3, 60, (b,), generator=gen, dtype=torch.int32))):
        outs = [torch.full((b, rows, g, d), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        fm.read_cache_fp8(*made, args[0], longer.cuda(), *outs, starts=on(starts))
        for n, out in enumerate(outs):
            want = torch.full((b, rows, g, d), 7.0, dtype=torch.float64)
            for i in range(b):
                first = 0 if starts is None else int(starts[i])
                for row in range(rows):
                    if 0 <= first + row < int(longer[i]):
                        page_of, slot = int(table[i, (first + row) // page]), (first + row) % page
                        code = expect[n][page_of, slot].long()
                        value = torch.where((code & 127) == 127, float("nan"), VALUES[(code & 127).clamp(max=126)]) * torch.where(code > 127, -1.0, 1.0)
                        want[i, row] = value * torch.pow(2.0, expect[2 + n][page_of, slot].double() - 127)[:, None]
            assert torch.equal(out.cpu().double().nan_to_num(nan=1e300), want.to(dtype).double().nan_to_num(nan=1e300))
    assert fm.device_status() == 0


@pytest.mark.parametrize("b,t,g,d,page", [(4, 2600, 8, 128, 40), (3, 9500, 8, 128, 16), (2, 21001, 5, 64, 7), (1, 4001, 100, 64, 64)])
def test_many_tokens_at_once_are_the_same_as_few_at_a_time(b, t, g, d, page):
    """Calls so large that a CTA has several rounds of tokens, against calls of 100 tokens; each sequence has one token fewer than the one before it."""
    per = -(-t // page)
    k, v = (x.cuda() for x in (data(b, t, g, d, torch.bfloat16, 1), data(b, t, g, d, torch.bfloat16, 2)))
    table = torch.randperm(b * per, generator=torch.Generator().manual_seed(t)).view(b, per).int().cuda()
    lengths, counts = torch.zeros(b, dtype=torch.int32, device="cuda"), t - torch.arange(b, dtype=torch.int32, device="cuda")
    at_once, one_by_one = cache(b * per, page, g, d), cache(b * per, page, g, d)
    fm.write_cache_fp8(k, v, *at_once, table, lengths, counts=counts)
    for i in range(0, t, 100):
        fm.write_cache_fp8(k[:, i:i + 100], v[:, i:i + 100], *one_by_one, table, lengths + i, counts=counts - i)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(at_once, one_by_one))
    outs, pieces = ([torch.full((b, t + 3, g, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2))
    fm.read_cache_fp8(*at_once, table, counts, *outs)
    for i in range(0, t + 3, 100):
        fm.read_cache_fp8(*at_once, table, counts, *(x[:, i:i + 100] for x in pieces), starts=torch.full_like(lengths, i))
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(outs, pieces)) and fm.device_status() == 0
    assert all((x[i, t - i:] == 7).all() for x in outs for i in range(b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_is_read_back_is_near_what_was_written(dtype):
    """Half a step of E4M3, 2^-4 of a value, or of its least step where a value is that much smaller than its head's largest; never infinite."""
    k = torch.randn((1, 512, 8, 128), generator=torch.Generator().manual_seed(3)).to(dtype)
    k[0, 0] = torch.finfo(dtype).max
    made = fm.make_cache_fp8(32, 16, 8, 128)
    table, zero = torch.arange(32, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda")
    fm.write_cache_fp8(k.cuda(), -k.cuda(), *made, table, zero)
    a, b = torch.zeros_like(k, device="cuda"), torch.zeros_like(k, device="cuda")
    fm.read_cache_fp8(*made, table, zero + 512, a, b)
    assert torch.equal(a, -b) and a.isfinite().all()
    k = k.double()
    step = torch.pow(2.0, made[2][table[0].long()].reshape(1, 512, 8, 1).cpu().double() - 127 - 9)
    assert ((a.cpu().double() - k).abs() <= torch.maximum(k.abs() * 2.0 ** -4, step / 2)).all()


def test_places_that_there_are_not():
    """Pages that do not exist, tokens that do not, places behind the table: nothing is written or read for them, all else is, and the status says so."""
    b, t, g, d, page = 3, 6, 2, 64, 4
    k, v = data(b, t, g, d, torch.float16, 1).cuda(), data(b, t, g, d, torch.float16, 2).cuda()
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4)
    lengths = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    good = cache(12, page, g, d)
    fm.write_cache_fp8(k, v, *good, table, lengths)
    assert fm.device_status() == 0
    for wrong in (-1, 12, 1 << 30, -(1 << 31)):
        bad_table = table.clone()
        bad_table[1, 1] = wrong                                    # the second sequence's tokens 4 .. 7
        made, start = cache(12, page, g, d), cache(12, page, g, d)
        fm.write_cache_fp8(k, v, *made, bad_table, lengths)
        assert fm.device_status() == 4
        for a, full, before in zip(made, good, start):
            a, full, before = (x.view(torch.uint8) for x in (a, full, before))
            assert torch.equal(a[:5], full[:5]) and torch.equal(a[6:], full[6:]) and torch.equal(a[5], before[5])
        outs = [torch.full((b, 9, g, d), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        fm.read_cache_fp8(*good, bad_table, lengths + 6, *outs)
        assert fm.device_status() == 4 and (outs[0][1, 4:8] == 5).all() and (outs[0][0, 7:] == 5).all() and not (outs[1][1, :4] == 5).all()
    # behind the table, of lengths that the table cannot hold, below zero (as zero)
    made, start = cache(12, page, g, d), cache(12, page, g, d)
    fm.write_cache_fp8(k, v, *made, table, torch.tensor([12, 1 << 30, -9], dtype=torch.int32, device="cuda"))
    assert fm.device_status() == 4
    for n, a, before in zip(itertools.count(), made, start):
        a, before = a.view(torch.uint8).view(48, *a.shape[2:]) if n < 2 else a.reshape(48, g), before.view(torch.uint8).view(48, *before.shape[2:]) if n < 2 else before.reshape(48, g)
        assert torch.equal(a[:12], before[:12]) and torch.equal(a[16:32], before[16:32]) and torch.equal(a[38:], before[38:])
        assert not torch.equal(a[12:16], before[12:16]) and not torch.equal(a[32:38], before[32:38])
    # token numbers
    made, start = cache(12, page, g, d), cache(12, page, g, d)
    fm.write_cache_fp8(k, v, *made, table, lengths, tokens=torch.tensor([[0, 6, 1], [-1, -5, -1], [1 << 30, 2, 5]], dtype=torch.int32, device="cuda"))
    assert fm.device_status() == 4
    one, two = (x[0].view(torch.uint8).view(48, g, d) for x in (made, start))
    kept = torch.tensor([i for i in range(48) if i not in (1, 3, 32 + 4, 32 + 5)], device="cuda")
    assert torch.equal(one[kept], two[kept]) and not torch.equal(one[36], two[36])


def test_strides_streams_and_graphs():
    b, t, g, d, page = 2, 9, 3, 128, 8
    k, v = data(b, t, g, d, torch.bfloat16, 1).cuda(), data(b, t, g, d, torch.bfloat16, 2).cuda()
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1))[:10].view(2, 5).int().cuda()
    lengths = torch.tensor([3, 20], dtype=torch.int32, device="cuda")
    one = cache(12, page, g, d)
    fm.write_cache_fp8(k, v, *one, table, lengths)
    # heads before slots, bytes by slot, values among others, keys and values as parts of one tensor
    two = cache(12, page, g, d)
    other = [two[0].transpose(1, 2).contiguous().transpose(1, 2), torch.cat([two[1].view(torch.uint8)] * 2, 3).view(torch.float8_e4m3fn)[..., :d], two[2].contiguous(),
             two[3].permute(2, 1, 0).contiguous().permute(2, 1, 0)]
    both = torch.cat([k, v], 2)
    wide_table = torch.cat([table, table], 1)[:, :5]
    fm.write_cache_fp8(both[:, :, :g], both[:, :, g:], *other, wide_table, lengths)
    for a, b_ in zip(one, other):
        assert torch.equal(a.contiguous().view(torch.uint8), b_.contiguous().view(torch.uint8))
    outs = [torch.zeros((b, 29, g, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    fm.read_cache_fp8(*one, table, lengths + t, *outs)
    split = torch.zeros((b, g, 29, 2 * d), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        fm.read_cache_fp8(*other, wide_table, lengths + t, split[..., :d], split[..., d:])
    stream.synchronize()
    assert all(torch.equal(x.view(torch.int16), y.contiguous().view(torch.int16)) for x, y in zip(outs, (split[..., :d], split[..., d:])))
    # one graph for any lengths, lists and counts
    made, tokens, counts = cache(12, page, g, d), torch.zeros((b, 4), dtype=torch.int32, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        fm.write_cache_fp8(k, v, *made, table, lengths, tokens=tokens, counts=counts)
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        lengths.copy_(torch.randint(0, 30, (b,), generator=gen))
        tokens.copy_(torch.randint(0, t, (b, 4), generator=gen))
        counts.copy_(torch.randint(0, 5, (b,), generator=gen))
        eager = [x.clone() for x in made]
        fm.write_cache_fp8(k, v, *eager, table, lengths, tokens=tokens, counts=counts)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(made, eager))
    assert fm.device_status() == 0


def test_long_cache_offsets():
    """A cache of more than 2^32 values, whose last page is written and read."""
    g, d, page = 8, 128, 128
    pages = (1 << 32) // (page * g * d) + 2
    made = fm.make_cache_fp8(pages, page, g, d)
    k, v = data(1, 200, g, d, torch.float16, 1).cuda(), data(1, 200, g, d, torch.float16, 2).cuda()
    table, zero = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    fm.write_cache_fp8(k, v, *made, table, zero)
    small = fm.make_cache_fp8(2, page, g, d)
    fm.write_cache_fp8(k, v, *small, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), zero)
    outs, expect = ([torch.zeros((1, 200, g, d), dtype=torch.float16, device="cuda") for _ in range(2)] for _ in range(2))
    fm.read_cache_fp8(*made, table, zero + 200, *outs)
    fm.read_cache_fp8(*small, table * 0 + torch.tensor([1, 0], dtype=torch.int32, device="cuda"), zero + 200, *expect)
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(outs, expect)) and fm.device_status() == 0
    assert not made[0][: pages - 2].view(torch.uint8).any()


def test_nothing_to_do_and_refusals():
    b, t, g, d = 2, 3, 2, 64
    k, v = torch.randn((b, t, g, d), device="cuda").half(), torch.randn((b, t, g, d), device="cuda").half()
    made = fm.make_cache_fp8(4, 8, g, d)
    table, lengths = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.zeros(2, dtype=torch.int32, device="cuda")
    names = ("k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "page_table", "lengths")
    good = dict(zip(names, (k, v, *made, table, lengths)))
    for call in (fm.write_cache_fp8, fm.read_cache_fp8):
        call(**good)
        call(**dict(good, k=k[:0], v=v[:0], page_table=table[:0], lengths=lengths[:0]))
        call(**dict(good, k=k[:, :0], v=v[:, :0]))
        none = dict(good, page_table=table[:, :0], **{n: good[n][:0] for n in names[2:6]})
        call(**none)
        assert fm.device_status() == (4 if call is fm.write_cache_fp8 else 0)      # tokens without a place
        for at, value in [("k", k.float()), ("k", k.cpu()), ("k", k[..., :32]), ("v", v[:, :2]), ("v", v.bfloat16()), ("v", v.cpu()), ("k_cache", made[0][:1]), ("k_cache", made[0].half()),
                          ("v_cache", made[1].cpu()), ("v_cache", made[1].view(torch.uint8)), ("k_scales", made[2].float()), ("k_scales", made[2][:, :4]), ("v_scales", made[3].cpu()),
                          ("page_table", table.long()), ("page_table", table[:1]), ("page_table", table.cpu()), ("page_table", table.t()), ("lengths", lengths.long()), ("lengths", lengths[:1]),
                          ("lengths", lengths.cpu()), ("k", k.transpose(2, 3).contiguous().transpose(2, 3)), ("k", torch.zeros((b, t, g, d + 4), device="cuda").half()[..., :d]), ("k", k[0])]:
            with pytest.raises(RuntimeError):
                call(**dict(good, **{at: value}))
    ints = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    for more in (dict(tokens=ints.long()), dict(tokens=ints[:1]), dict(tokens=ints.cpu()), dict(tokens=ints[0]), dict(tokens=ints.t().contiguous().t()), dict(counts=ints), dict(counts=lengths.long()), dict(counts=lengths.cpu())):
        with pytest.raises(RuntimeError):
            fm.write_cache_fp8(**good, **more)
    for more in (dict(starts=ints), dict(starts=lengths.long()), dict(starts=lengths.cpu())):
        with pytest.raises(RuntimeError):
            fm.read_cache_fp8(**good, **more)
    # tensors that are written whose places share memory
    for at, value in (("k_cache", made[0][:1].expand(4, 8, g, d)), ("v_scales", made[3][:, :1].expand(4, 8, g))):
        with pytest.raises(RuntimeError):
            fm.write_cache_fp8(**dict(good, **{at: value}))
    with pytest.raises(RuntimeError):
        fm.read_cache_fp8(**dict(good, k=k[:1].expand(b, t, g, d)))
