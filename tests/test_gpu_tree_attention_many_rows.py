"""tree_attention with more than 32 rows (drafted tokens times heads of queries) per head of keys: what masks, pages, strides and
values that are not finite do there.  Bounds are those of test_gpu_tree_attention.py."""
import pytest
import torch

import fp6_marlin_b200 as fm
from test_gpu_tree_attention import _check, _inputs, _run

pytestmark = pytest.mark.gpu

# tokens, heads, heads of keys, values of a head: up to 64 rows, up to 128, two row tiles, three
SHAPES = [(12, 4, 1, 128), (20, 8, 2, 64), (31, 8, 2, 128), (50, 8, 2, 64), (64, 8, 2, 128), (33, 8, 1, 64), (40, 32, 4, 128)]
# tokens of a page: whole runs by TMA (a tile, part of one, several), single tokens
PAGES = [64, 16, 24, 256, 12, 1]


def _without(x, gone):
    """x with a cache of single tokens from which the tokens of the pages `gone` (sequence, place in the table) are missing."""
    page = x["k_cache"].shape[1]
    kept = []
    for i, n in enumerate(x["lengths"].tolist()):
        at = torch.arange(n, device="cuda")
        for row, place in gone:
            if row == i:
                at = at[at // page != place]
        kept.append((x["page_table"][i].long()[at // page], at % page))
    y = dict(x, lengths=torch.tensor([len(rows) for rows, _ in kept], dtype=torch.int32, device="cuda"))
    rows, slots = (torch.cat([pair[e] for pair in kept]) for e in (0, 1))
    y["k_cache"], y["v_cache"] = x["k_cache"][rows, slots][:, None], x["v_cache"][rows, slots][:, None]
    ends = y["lengths"].cumsum(0)
    y["page_table"] = ((ends - y["lengths"])[:, None] + torch.arange(max(1, int(y["lengths"].max())), device="cuda")).clamp(max=max(len(rows) - 1, 0)).int()
    return y


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("page", PAGES)
def test_pages_that_do_not_exist(t, h, g, d, page):
    """Their tokens are hidden and the status says so: the first page, one in the middle, the last (of a partial tile), a whole sequence's."""
    lengths = [700, 64, 1111, 5]
    x = _inputs(4, t, h, g, d, lengths, page)
    expect = _run(x)
    assert fm.device_status() == 0
    places = [-(-n // page) for n in lengths]
    gone = [(0, 0), (0, places[0] // 2), (2, places[2] - 1), (2, places[2] // 3), *((3, i) for i in range(places[3]))]
    good = x["page_table"].clone()
    for wrong in (-1, x["k_cache"].shape[0], 1 << 30, -(1 << 31)):
        for row, place in gone:
            x["page_table"][row, place] = wrong
        out = _run(x)
        assert fm.device_status() == 4
        assert torch.equal(out, _run(x)) and fm.device_status() == 4
    _check(out, _without(dict(x, page_table=good), gone))
    x["page_table"].copy_(good)
    assert torch.equal(_run(x), expect) and fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", [(12, 16, 4, 128), (40, 16, 2, 64)])
def test_heads_that_share_memory(t, h, g, d):
    """One head of keys and values for all, and one page for all places of the table."""
    x = _inputs(2, t, h, g, d, [150, 700], 16)
    for n in ("k_cache", "v_cache", "k", "v"):
        x[n] = x[n][:, :, :1].expand_as(x[n])
    _check(_run(x), x)
    for n in ("k_cache", "v_cache"):
        x[n] = x[n][3:4].expand_as(x[n])
    _check(_run(x), x)
    assert fm.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [33, 36, 63, 64, 65, 100, 127, 128, 129, 192, 256, 257, 320, 384, 511, 512])
def test_rows_of_a_head_of_keys(rows, dtype):
    """Row tiles that are full, nearly empty, odd in number; sequences from none to several key tiles."""
    group = next((n for n in (8, 7, 4, 3, 5, 1) if rows % n == 0 and rows // n <= 64), None)
    t, h, g = (rows // group, 2 * group, 2) if group else (1, rows, 1)
    x = _inputs(5, t, h, g, 64 if rows % 2 else 128, [0, 63, 64, 129, 700], 16, dtype, fill=float("nan"))
    out = _run(x)
    _check(out, x)
    assert torch.equal(out, _run(x)) and fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", [(9, 16, 4, 128), (25, 8, 2, 64), (33, 8, 1, 128)])
@pytest.mark.parametrize("page", [64, 8, 5])
def test_many_lengths(t, h, g, d, page):
    x = _inputs(41, t, h, g, d, list(range(0, 41 * 9, 9)), page, fill=float("inf"))
    _check(_run(x), x)
    assert fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("lengths,page", [([0, 0], 16), ([200, 0], 64), ([65, 1300], 16), ([65, 1300], 12), ([2000, 129], 128)])
def test_padding_and_rows_that_see_nothing(t, h, g, d, lengths, page):
    x = _inputs(2, t, h, g, d, lengths, page, fill=float("inf"))
    x["tree"][0, 2], x["tree"][1, 3:] = 0, 0
    x["tree"][1, 0] = 0b010                                        # sees another token, not itself
    x["tree"][0] &= ~0b100
    x["tree"][1] &= 0b111
    x["k"][0, 2], x["v"][0, 2] = float("nan"), float("nan")        # what padding holds is seen by nobody
    x["k"][1, 3:], x["v"][1, 3:] = float("inf"), float("-inf")
    x["q"][0, 2], x["q"][1, 4] = float("nan"), float("inf")
    out = _run(x)
    assert (out[0, 2] == 0).all() and (out[1, 3:] == 0).all()
    clean = {n: v.clone() for n, v in x.items()}
    for n in ("q", "k", "v"):
        clean[n][0, 2], clean[n][1, 3:] = 0, 0
    _check(out, clean)
    x["tree"][:] = 0                                               # nothing but padding
    assert (_run(x) == 0).all() and fm.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("length", [0, 40, 64, 700, 6000])
def test_values_that_are_not_finite_reach_those_that_see_them(t, h, g, d, length, dtype):
    """Token 1 sees token 0 and itself, the others only themselves; token 0's values hold an infinity and a NaN, the last token's a negative infinity."""
    x = _inputs(1, t, h, g, d, [length], 16, dtype)
    x["tree"] = 1 << torch.arange(t, device="cuda")
    x["tree"][1] = 0b11
    spots = [(0, 5, float("inf")), (0, 7, float("nan")), (t - 1, d - 1, float("-inf"))]
    for token, column, value in spots:
        x["v"][0, token, 0, column] = value
    out = _run(x).float()
    heads = slice(0, h // g)
    assert out[0, :2, heads, 5].isposinf().all() and out[0, :2, heads, 7].isnan().all() and out[0, t - 1, heads, d - 1].isneginf().all()
    clean = {n: v.clone() for n, v in x.items()}
    for token, column, _ in spots:
        clean["v"][0, token, 0, column] = 0
    rest = _run(clean)
    out[0, :2, heads, 5], out[0, :2, heads, 7], out[0, t - 1, heads, d - 1] = rest[0, :2, heads, 5].float(), rest[0, :2, heads, 7].float(), rest[0, t - 1, heads, d - 1].float()
    assert out.isfinite().all()
    _check(out.to(dtype), clean)


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("page", [16, 12])
def test_one_mask_for_all_and_strided_tensors(t, h, g, d, page):
    x = _inputs(3, t, h, g, d, [150, 0, 1333], page)
    x["tree"] = chain = fm.tree_masks(torch.arange(t) - 1).cuda()
    one = _run(x)
    _check(one, x)
    # heads first, the cache's heads before its slots, its values among others, a page table and masks with longer rows
    y = dict(x)
    y["q"] = x["q"].transpose(1, 2).contiguous().transpose(1, 2)
    y["k"], y["v"] = x["k"].transpose(0, 1).contiguous().transpose(0, 1), x["v"].contiguous()
    y["k_cache"] = x["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    y["v_cache"] = torch.cat([x["v_cache"], x["v_cache"]], 3)[..., :d]
    y["page_table"] = torch.cat([x["page_table"], torch.full((3, 2), 1 << 30, dtype=torch.int32, device="cuda")], 1)[:, : x["page_table"].shape[1]]
    y["tree"] = torch.cat([chain.expand(3, t), torch.zeros((3, 1), dtype=torch.int64, device="cuda")], 1)[:, :t]
    out = torch.zeros((3, h, t, d), dtype=torch.float16, device="cuda").transpose(1, 2)
    names = ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")
    fm.tree_attention(*(y[n] for n in names), out)
    assert torch.equal(out, one)
    # the same memory under other strides: the slots of two caches in turn, then every other page
    both = torch.stack([x["k_cache"], x["v_cache"]], 2).flatten(1, 2)
    y["k_cache"], y["v_cache"] = both[:, 0::2], both[:, 1::2]
    assert torch.equal(_run(y), one)
    y["k_cache"], y["v_cache"] = (torch.stack([x[n], torch.full_like(x[n], float("nan"))], 1).flatten(0, 1)[::2] for n in ("k_cache", "v_cache"))
    assert torch.equal(_run(y), one)
    assert fm.device_status() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_strides_of_single_places(d):
    """One sequence, one token, one head of keys, one page: whatever their strides are."""
    x = _inputs(1, 1, 48, 1, d, [9], 16, spare=0)
    expect = _run(x)
    _check(expect, x)
    for n, at in (("k", (0, 1, 2)), ("v", (0, 1, 2)), ("k_cache", (0, 2)), ("v_cache", (0, 2)), ("q", (0, 1))):
        x[n] = x[n].contiguous().as_strided(x[n].shape, [1 if i in at else s for i, s in enumerate(x[n].stride())])
    assert torch.equal(_run(x), expect)


@pytest.mark.parametrize("t,h,g,d", SHAPES)
def test_lengths_out_of_range(t, h, g, d):
    x = _inputs(3, t, h, g, d, [300, 48, 480], 16)
    same = {n: v.clone() for n, v in x.items()}
    x["lengths"] = torch.tensor([1 << 30, -5, 480], dtype=torch.int32, device="cuda")     # cut to the table, to zero
    same["lengths"] = torch.tensor([480, 0, 480], dtype=torch.int32, device="cuda")
    out = _run(x)
    _check(out, same)
    assert torch.equal(out, _run(same)) and fm.device_status() == 0


@pytest.mark.parametrize("t", [10, 40])
@pytest.mark.parametrize("page", [128, 4])
def test_long_cache_offsets(t, page):
    """A cache of more than 2^31 values, whose last pages are used."""
    g, d = 8, 128
    pages = (1 << 31) // (page * g * d) + 1024 // page + 1
    kc = torch.zeros((pages, page, g, d), dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    x = _inputs(1, t, 32, g, d, [1000], page)
    table = torch.arange(pages - x["page_table"].shape[1], pages, device="cuda").flip(0)[None].int()
    kc[table[0].long()], vc[table[0].long()] = x["k_cache"][x["page_table"][0].long()], x["v_cache"][x["page_table"][0].long()]
    expect = _run(x)
    _check(expect, x)
    x["k_cache"], x["v_cache"], x["page_table"] = kc, vc, table
    assert torch.equal(_run(x), expect)


@pytest.mark.parametrize("t,h,g,d", [(20, 8, 2, 64), (40, 32, 4, 128)])
def test_streams_and_graph(t, h, g, d):
    sets = [_inputs(2, t, h, g, d, [3000, 1000 + seed], 16, seed=seed) for seed in (1, 2)]
    expect = [_run(x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = _run(sets[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, expect))
    graph, x, out = torch.cuda.CUDAGraph(), sets[0], torch.zeros_like(expect[0])
    names = ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")
    with torch.cuda.graph(graph, stream=streams[0]):
        fm.tree_attention(*(x[n] for n in names), out)
    for n in (3000, 7, 0, 2999, 64):                               # lengths are the device's: one graph serves all
        x["lengths"][0] = n
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x)
    assert fm.device_status() == 0
