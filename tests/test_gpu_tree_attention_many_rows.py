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
