"""tree_attention_fp8 against softmax attention in 64 bits over the values that the cache stands for.

Bounds, with u = 2^-11 (fp16) or 2^-8 (bf16): the result is rounded once (u of itself); the weights, times their values' powers of two, are rounded once to fp16 (w = 2^-11,
at most w = u where a head of keys has more than 32 rows) before they meet the E4M3 values: w of sum p |v|, and as much again where their sum is taken of the
unrounded ones.  Weights are relative to the largest of a row, max p_j 2^y_j, and multiples of 2^-24 at least: 2^-25 * max_j (p_j 2^y_j) * sum_j |v_j| 2^-y_j; where a head of keys has
more than 32 rows the values come times their powers and the weights are p_j alone: in fp16 each is off by up to 2^-25 * max_j p_j, which is 2^-25 * max_j p_j * sum_j |v_j|.  Scores are fp32
sums of D products, each addition off by at most 2^-23: D * 2^-23 * scale * sum |q k| in the exponent; the exponent, a score in powers of two and y, is rounded twice, and so is the
maximum that is taken from it: 4 * 2^-24 * (their largest magnitude); all of that twice (weight and total), plus 2^-20 for the exponentials and the running sums.
"""
import math

import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu

BITS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
NAMES = ("q", "k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "page_table", "lengths", "tree")


def _bytes(t):
    return t.view(torch.uint8)


def inputs(b, t, h, g, d, lengths, page, dtype=torch.float16, seed=0, spare=2, fill=None, spread=1.0):
    """Caches of E4M3 values of unit size with exponents that differ from token to token and head to head (`spread`: their deviation in powers of two)."""
    gen = torch.Generator(device="cuda").manual_seed(seed + b + 3 * t + 5 * h + 7 * d + 11 * page)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    per = max(1, -(-int(lengths.max()) // page))
    pages = b * per + spare
    qkv = torch.randn((b, t, (h + 2 * g) * d), generator=gen, device="cuda").to(dtype)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: b * per].view(b, per).int().cuda()
    parents = torch.tensor([[(i * 7 + r) % (i + 1) - 1 for i in range(t)] for r in range(b)])
    x = {"q": qkv[..., : h * d].unflatten(2, (h, d)), "k": qkv[..., h * d:(h + g) * d].unflatten(2, (g, d)), "v": qkv[..., (h + g) * d:].unflatten(2, (g, d)),
         "page_table": table, "lengths": lengths.cuda(), "tree": fm.tree_masks(parents).cuda()}
    for n in ("k", "v"):
        x[n + "_cache"] = (100 * torch.randn((pages, page, g, d), generator=gen, device="cuda")).clamp(-448, 448).to(torch.float8_e4m3fn)
        power = (-7 + spread * torch.randn((pages, g, page), generator=gen, device="cuda")).round().clamp(-15, 8)
        x[n + "_scales"] = (power + 127).to(torch.uint8).transpose(1, 2)
        # (as written from fp16: 448 * 2^8 is none of its values)
        x[n + "_cache"] = x[n + "_cache"].float().clamp(-240, 240).where(x[n + "_scales"][..., None] == 127 + 8, x[n + "_cache"].float()).to(torch.float8_e4m3fn)
    if fill is not None:          # what must not be read: slots behind the last token, pages of nobody
        used = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
        for i, n in enumerate(lengths.tolist()):
            at = torch.arange(n, device="cuda")
            used[table[i].long()[at // page], at % page] = True
        for n in ("k", "v"):
            _bytes(x[n + "_cache"])[~used] = 0x7f                    # NaN
            x[n + "_scales"][~used] = fill
    return x


def tokens(x, name, i, at):
    """The values of tokens `at` of sequence i, and their powers of two, in 64 bits."""
    page = x[name + "_cache"].shape[1]
    rows, slots = x["page_table"][i].long()[at // page], at % page
    power = torch.pow(2.0, x[name + "_scales"][rows, slots].double() - 127)
    return _bytes(x[name + "_cache"])[rows, slots].view(torch.float8_e4m3fn).double() * power[..., None], power


def exact(x, scale=None):
    """The result and the bound of its error."""
    q, k, v, tree = x["q"].double(), x["k"].double(), x["v"].double(), x["tree"].cpu()
    b, t, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    group, u = h // k.shape[2], BITS[x["q"].dtype]
    w = u if t * group > 32 else 2.0 ** -11
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    # the powers of drafted values: fp16 as they are, bf16 so that the largest of a head is below 2^15
    own = torch.ones(v.shape[:3], dtype=torch.float64, device="cuda")
    if x["q"].dtype == torch.bfloat16:
        own = torch.pow(2.0, torch.floor(torch.log2(v.nan_to_num(0, 0, 0).abs().amax(3).clamp(min=2.0 ** -86))) - 14)
    for i, n in enumerate(x["lengths"].tolist()):
        at = torch.arange(n, device="cuda")
        (keys, _), (values, powers) = tokens(x, "k", i, at), tokens(x, "v", i, at)
        keys, values = (torch.cat(pair).repeat_interleave(group, 1) for pair in ((keys, k[i]), (values, v[i])))              # n + t, h, d
        powers = torch.cat([powers, own[i]]).repeat_interleave(group, 1)
        for j in range(t):
            word = int(tree[j] if tree.dim() == 1 else tree[i, j])
            if word == 0:
                continue
            seen = torch.tensor([True] * n + [bool(word >> c & 1) for c in range(t)], device="cuda")
            if not seen.any():
                continue
            ks, vs, ps = keys[seen], values[seen], powers[seen]
            s = torch.einsum("hd,nhd->hn", q[i, j], ks) * scale
            p = torch.softmax(s, 1)
            out[i, j] = torch.einsum("hn,nhd->hd", p, vs)
            size = torch.einsum("hn,nhd->hd", p, vs.abs())
            slack = (torch.einsum("hd,nhd->hn", q[i, j].abs(), ks.abs()) * abs(scale)).amax(1, keepdim=True) * d * 2.0 ** -23
            largest = (s.abs() / math.log(2) + torch.log2(ps.T).abs()).amax(1, keepdim=True)
            many = t * group > 32
            least = 2.0 ** -25 * (p if many else p * ps.T).amax(1, keepdim=True) * (vs.abs() / (1 if many else ps[..., None])).sum(0)
            bound[i, j] = u * out[i, j].abs() + (2 * w + 2 * slack + 8 * 2.0 ** -24 * largest + 2.0 ** -20) * size + least + 2.0 ** -25
    return out, bound


def run(x, **more):
    out = torch.full(x["q"].shape, float("nan"), dtype=x["q"].dtype, device="cuda")
    fm.tree_attention_fp8(*(x[n] for n in NAMES), out, **more)
    return out


def check(out, x, scale=None):
    expect, bound = exact(x, scale)
    err = (out.double() - expect).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


CASES = [
    # b, t, heads, kv heads, d, lengths, page (up to 16 rows of a head of keys, up to 32, more; whole runs of a page and single tokens)
    (1, 1, 1, 1, 128, [0], 16), (1, 1, 32, 32, 128, [1], 16), (1, 1, 32, 32, 128, [300], 16), (1, 1, 8, 1, 64, [127], 16), (1, 1, 8, 1, 64, [128], 16), (2, 1, 8, 8, 64, [129, 0], 1),
    (3, 5, 32, 8, 128, [0, 1000, 17], 16), (1, 64, 64, 8, 128, [500], 48), (2, 64, 8, 8, 64, [129, 2048], 64), (1, 16, 1, 1, 128, [4097], 24), (2, 17, 1, 1, 64, [255, 256], 24),
    (4, 7, 10, 2, 128, [5, 6, 7, 8], 3), (2, 33, 9, 3, 64, [100, 31], 7), (1, 3, 64, 1, 128, [1025], 256), (5, 2, 4, 4, 128, [900, 3, 64, 128, 127], 128), (1, 32, 1, 1, 64, [600], 16),
    (17, 4, 16, 2, 128, list(range(0, 17 * 40, 40)), 16), (1, 1, 64, 8, 128, [20000], 16), (1, 64, 32, 4, 128, [9000], 16), (70, 1, 8, 2, 64, [i * 5 for i in range(70)], 32),
    (1, 17, 8, 8, 128, [777], 4096), (3, 64, 3, 1, 128, [64, 0, 200], 16), (2, 8, 8, 2, 128, [383, 1], 8), (1, 1, 71, 1, 128, [900], 16), (1, 31, 3, 3, 64, [513], 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,g,d,lengths,page", CASES)
def test_attention(b, t, h, g, d, lengths, page, dtype):
    x = inputs(b, t, h, g, d, lengths, page, dtype, fill=255)
    for _ in range(2):
        out = run(x)
        check(out, x)
    assert torch.equal(out, run(x)) and fm.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 4, 5, 15, 16, 17, 31, 32, 33, 36, 63, 64, 65, 100, 127, 128, 129, 192, 256, 257, 320, 384, 511, 512])
def test_rows_of_a_head_of_keys(rows, dtype):
    """Row tiles that are full, nearly empty, odd in number; sequences from none to several key tiles."""
    group = next((n for n in (8, 7, 4, 3, 5, 1) if rows % n == 0 and rows // n <= 64), None)
    t, h, g = (rows // group, 2 * group, 2) if group else (1, rows, 1)
    x = inputs(5, t, h, g, 64 if rows % 2 else 128, [0, 127, 128, 257, 1400], 16, dtype, fill=0)
    out = run(x)
    check(out, x)
    assert torch.equal(out, run(x)) and fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", [(1, 4, 1, 128), (8, 32, 4, 128), (7, 8, 1, 64), (16, 8, 1, 128), (40, 8, 2, 64), (9, 2, 1, 128)])
def test_rows_joined_from_many_ranges(t, h, g, d):
    """One long sequence and few heads of keys: every multiprocessor leaves a part of the same rows; few and many rows after one another."""
    x, other = inputs(1, t, h, g, d, [24690], 16, torch.bfloat16), inputs(1, 3, 2, 1, d, [8642], 16, torch.bfloat16)
    first, first_other = run(x), run(other)
    check(first, x)
    check(first_other, other)
    for _ in range(5):
        assert torch.equal(run(x), first) and torch.equal(run(other), first_other)
    x["v"][0, 0, 0, 3] = float("inf")                                # it reaches the rows that see it through the joined parts as well
    heads = h // g
    out, sees = run(x)[0].float(), (x["tree"].reshape(-1) & 1).bool()
    assert (out[:, :heads, 3].isposinf() == sees[:, None]).all() and out[~sees].isfinite().all() and fm.device_status() == 0


SHAPES = [(1, 4, 1, 128), (6, 8, 2, 128), (3, 16, 2, 64), (12, 4, 1, 128), (20, 8, 2, 64), (50, 8, 2, 64), (64, 8, 2, 128), (40, 32, 4, 128)]


@pytest.mark.parametrize("t,h,g,d", SHAPES[1:])
@pytest.mark.parametrize("lengths", [[0, 0], [200, 0], [65, 1300], [128, 129]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_padding_and_rows_that_see_nothing(t, h, g, d, lengths, dtype):
    x = inputs(2, t, h, g, d, lengths, 16, dtype, fill=254)
    x["tree"][0, 2], x["tree"][1, min(t - 1, 3):] = 0, 0
    x["tree"][1, 0] = 0b010                                        # sees another token, not itself
    x["tree"][0] &= ~0b100
    x["tree"][1] &= (1 << min(t - 1, 3)) - 1
    last = min(t - 1, 3)
    x["k"][0, 2], x["v"][0, 2] = float("nan"), float("nan")        # what padding holds is seen by nobody
    x["k"][1, last:], x["v"][1, last:] = float("inf"), float("-inf")
    x["q"][0, 2], x["q"][1, last] = float("nan"), float("inf")
    out = run(x)
    assert (out[0, 2] == 0).all() and (out[1, last:] == 0).all()
    clean = {n: v.clone() for n, v in x.items()}
    for n in ("q", "k", "v"):
        clean[n][0, 2], clean[n][1, last:] = 0, 0
    check(out, clean)
    x["tree"][:] = 0                                               # nothing but padding
    assert (run(x) == 0).all() and fm.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,h,g,d", SHAPES[1:])
@pytest.mark.parametrize("length", [0, 40, 128, 700, 6000])
def test_values_that_are_not_finite_reach_those_that_see_them(t, h, g, d, length, dtype):
    """Token 1 sees token 0 and itself, the others only themselves; token 0's values hold an infinity and a NaN, the last token's a negative infinity."""
    x = inputs(1, t, h, g, d, [length], 16, dtype)
    x["tree"] = 1 << torch.arange(t, device="cuda")
    x["tree"][1] = 0b11
    spots = [(0, 5, float("inf")), (0, 7, float("nan")), (t - 1, d - 1, float("-inf"))]
    for token, column, value in spots:
        x["v"][0, token, 0, column] = value
    out = run(x).float()
    heads = slice(0, h // g)
    assert out[0, :2, heads, 5].isposinf().all() and out[0, :2, heads, 7].isnan().all() and out[0, t - 1, heads, d - 1].isneginf().all()
    clean = {n: v.clone() for n, v in x.items()}
    for token, column, _ in spots:
        clean["v"][0, token, 0, column] = 0
    rest = run(clean)
    out[0, :2, heads, 5], out[0, :2, heads, 7], out[0, t - 1, heads, d - 1] = rest[0, :2, heads, 5].float(), rest[0, :2, heads, 7].float(), rest[0, t - 1, heads, d - 1].float()
    assert out.isfinite().all()
    check(out.to(dtype), clean)


def _without(x, gone):
    """x with a cache of single tokens from which the tokens of the pages `gone` (sequence, place in the table) are missing."""
    page, kept = x["k_cache"].shape[1], []
    for i, n in enumerate(x["lengths"].tolist()):
        at = torch.arange(n, device="cuda")
        for row, place in gone:
            if row == i:
                at = at[at // page != place]
        kept.append((x["page_table"][i].long()[at // page], at % page))
    y = dict(x, lengths=torch.tensor([len(rows) for rows, _ in kept], dtype=torch.int32, device="cuda"))
    rows, slots = (torch.cat([pair[e] for pair in kept]) for e in (0, 1))
    for n in ("k", "v"):
        y[n + "_cache"], y[n + "_scales"] = _bytes(x[n + "_cache"])[rows, slots][:, None].view(torch.float8_e4m3fn), x[n + "_scales"][rows, slots][:, None]
    ends = y["lengths"].cumsum(0)
    y["page_table"] = ((ends - y["lengths"])[:, None] + torch.arange(max(1, int(y["lengths"].max())), device="cuda")).clamp(max=max(len(rows) - 1, 0)).int()
    return y


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("page", [64, 16, 24, 256, 12, 1])
def test_pages_that_do_not_exist(t, h, g, d, page):
    """Their tokens are hidden and the status says so: the first page, one in the middle, the last (of a partial tile), a whole sequence's."""
    lengths = [700, 64, 1111, 5]
    x = inputs(4, t, h, g, d, lengths, page)
    expect = run(x)
    assert fm.device_status() == 0
    places = [-(-n // page) for n in lengths]
    gone = [(0, 0), (0, places[0] // 2), (2, places[2] - 1), (2, places[2] // 3), *((3, i) for i in range(places[3]))]
    good = x["page_table"].clone()
    for wrong in (-1, x["k_cache"].shape[0], 1 << 30, -(1 << 31)):
        for row, place in gone:
            x["page_table"][row, place] = wrong
        out = run(x)
        assert fm.device_status() == 4
        assert torch.equal(out, run(x)) and fm.device_status() == 4
    check(out, _without(dict(x, page_table=good), gone))
    x["page_table"].copy_(good)
    assert torch.equal(run(x), expect) and fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_scores_and_scale(t, h, g, d, dtype):
    """Scores in the thousands: the running maximum keeps every exponential in range."""
    x = inputs(2, t, h, g, d, [300, 70], 16, dtype)
    x["q"] = x["q"] * 30
    x["k_scales"] += 5
    for scale in (1.0, -0.5, 0.0):
        check(run(x, scale=scale), x, scale)


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_powers_of_two_that_differ(t, h, g, d, dtype):
    """Tokens whose values are thousands of times larger or smaller than others', tokens of zeros."""
    x = inputs(2, t, h, g, d, [900, 70], 16, dtype, spread=5.0)
    x["v"][:, 0] *= 2.0 ** -9
    _bytes(x["v_cache"])[:, 3::7], x["v_scales"][:, 3::7] = 0, 127 + (-15 if dtype == torch.float16 else -40)
    check(run(x), x)
    x["v"][:] = 0
    check(run(x), x)
    if dtype == torch.bfloat16:                                    # what fp16 does not hold
        x = inputs(2, t, h, g, d, [900, 70], 16, dtype)
        for n in ("v", "v_cache", "v_scales"):
            x[n] = x[n] + 50 if n == "v_scales" else x[n] * 2.0 ** 50 if n == "v" else x[n]
        x["q"], x["k_scales"], x["k"] = x["q"] * 2.0 ** 40, x["k_scales"] - 40, x["k"] * 2.0 ** -40
        check(run(x), x)


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("page", [16, 12])
def test_one_mask_for_all_and_strided_tensors(t, h, g, d, page):
    x = inputs(3, t, h, g, d, [150, 0, 1333], page)
    x["tree"] = chain = fm.tree_masks(torch.arange(t) - 1).cuda()
    one = run(x)
    check(one, x)
    # heads first, the cache's heads before its slots, its values among others, a page table and masks with longer rows
    y = dict(x)
    y["q"] = x["q"].transpose(1, 2).contiguous().transpose(1, 2)
    y["k"], y["v"] = x["k"].transpose(0, 1).contiguous().transpose(0, 1), x["v"].contiguous()
    y["k_cache"] = x["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    y["v_cache"] = torch.cat([_bytes(x["v_cache"])] * 2, 3)[..., :d].view(torch.float8_e4m3fn)
    y["k_scales"] = x["k_scales"].contiguous()
    y["v_scales"] = x["v_scales"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    y["page_table"] = torch.cat([x["page_table"], torch.full((3, 2), 1 << 30, dtype=torch.int32, device="cuda")], 1)[:, : x["page_table"].shape[1]]
    y["tree"] = torch.cat([chain.expand(3, t), torch.zeros((3, 1), dtype=torch.int64, device="cuda")], 1)[:, :t]
    out = torch.zeros((3, h, t, d), dtype=torch.float16, device="cuda").transpose(1, 2)
    fm.tree_attention_fp8(*(y[n] for n in NAMES), out)
    assert torch.equal(out, one)
    # the same memory under other strides: the slots of two caches in turn, then every other page
    both = torch.stack([_bytes(x["k_cache"]), _bytes(x["v_cache"])], 2).flatten(1, 2).view(torch.float8_e4m3fn)
    y["k_cache"], y["v_cache"] = both[:, 0::2], both[:, 1::2]
    assert torch.equal(run(y), one)
    # one power for a page, for all
    for n in ("k_scales", "v_scales"):
        x[n], y[n] = (z[:, :1].expand(x[n].shape) for z in (x[n], x[n].contiguous()))
    assert torch.equal(run(y), run(x))
    check(run(y), y)
    assert fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", [(1, 8, 4, 128), (12, 16, 4, 128), (40, 16, 2, 64)])
def test_heads_and_pages_that_share_memory(t, h, g, d):
    """One head of keys and values for all, and one page for all places of the table."""
    x = inputs(2, t, h, g, d, [150, 700], 16)
    for n in ("k_cache", "v_cache", "k", "v"):
        x[n] = x[n][:, :, :1].expand_as(x[n])
    check(run(x), x)
    for n in ("k_cache", "v_cache"):
        x[n] = x[n][3:4].expand_as(x[n])
    check(run(x), x)
    assert fm.device_status() == 0


@pytest.mark.parametrize("h,d", [(4, 64), (4, 128), (48, 64), (48, 128)])
def test_strides_of_single_places(h, d):
    """One sequence, one token, one head of keys, one page: whatever their strides are."""
    x = inputs(1, 1, h, 1, d, [9], 16, spare=0)
    expect = run(x)
    check(expect, x)
    for n, at in (("k", (0, 1, 2)), ("v", (0, 1, 2)), ("k_cache", (0, 2)), ("v_cache", (0, 2)), ("k_scales", (0, 2)), ("q", (0, 1))):
        steps = [1 if i in at else s for i, s in enumerate((x[n].contiguous()).stride())]
        x[n] = x[n].contiguous().as_strided(x[n].shape, steps)
    x["lengths"], x["page_table"], x["tree"] = x["lengths"].as_strided((1,), (5,)), x["page_table"].as_strided((1, 1), (4, 6)), x["tree"].as_strided((1, 1), (3, 7))
    assert torch.equal(run(x), expect)


@pytest.mark.parametrize("t,h,g,d", SHAPES)
def test_lengths_out_of_range_and_bits_behind_the_last_token(t, h, g, d):
    x = inputs(3, t, h, g, d, [300, 48, 480], 16)
    same = {n: v.clone() for n, v in x.items()}
    x["lengths"] = torch.tensor([1 << 30, -5, 480], dtype=torch.int32, device="cuda")     # cut to the table, to zero
    same["lengths"] = torch.tensor([480, 0, 480], dtype=torch.int32, device="cuda")
    expect = run(same)
    check(expect, same)
    assert torch.equal(run(x), expect)
    if t < 64:                                                     # they stand for no token; an entry that has only such bits sees the committed tokens
        x["tree"] |= -1 << t
        assert torch.equal(run(x), expect)
        x["tree"][:, t // 2] = 1 << t if t < 63 else -(1 << 63)
        x["lengths"] = same["lengths"]
        check(run(x), x)
    assert fm.device_status() == 0


@pytest.mark.parametrize("t", [1, 10, 40])
@pytest.mark.parametrize("page", [128, 4])
def test_long_cache_offsets(t, page):
    """A cache of more than 2^32 values, whose last pages are used."""
    g, d = 8, 128
    pages = (1 << 32) // (page * g * d) + 1024 // page + 1
    x = inputs(1, t, 32, g, d, [1000], page)
    expect = run(x)
    check(expect, x)
    table = torch.arange(pages - x["page_table"].shape[1], pages, device="cuda").flip(0)[None].int()
    for n in ("k_cache", "v_cache", "k_scales", "v_scales"):
        big = torch.zeros((pages, *x[n].shape[1:]), dtype=torch.uint8, device="cuda")
        big[table[0].long()] = _bytes(x[n].contiguous())[x["page_table"][0].long()]
        x[n] = big.view(x[n].dtype)
    x["page_table"] = table
    assert torch.equal(run(x), expect)


@pytest.mark.parametrize("t,h,g,d", [(1, 32, 8, 128), (5, 32, 8, 128), (20, 8, 2, 64), (40, 32, 4, 128)])
def test_streams_and_graph(t, h, g, d):
    sets = [inputs(2, t, h, g, d, [6000, 2000 + seed], 16, seed=seed) for seed in (1, 2)]
    expect = [run(x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = run(sets[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, expect))
    graph, x, out = torch.cuda.CUDAGraph(), sets[0], torch.zeros_like(expect[0])
    with torch.cuda.graph(graph, stream=streams[0]):
        fm.tree_attention_fp8(*(x[n] for n in NAMES), out)
    for n in (6000, 7, 0, 2999, 128):                              # lengths are the device's: one graph serves all
        x["lengths"][0] = n
        graph.replay()
        torch.cuda.synchronize()
        check(out, x)
    assert fm.device_status() == 0


def test_nothing_to_do_and_refusals():
    x = inputs(2, 3, 8, 2, 128, [20, 30], 16)
    good, out = [x[n] for n in NAMES], torch.empty_like(x["q"].contiguous())

    def call(at=None, value=None, o=out):
        args = list(good)
        if at is not None:
            args[NAMES.index(at)] = value
        fm.tree_attention_fp8(*args, o)

    call()
    rest = [x[n] for n in NAMES[3:7]]
    fm.tree_attention_fp8(x["q"][:0], x["k"][:0], x["v"][:0], *rest, x["page_table"][:0], x["lengths"][:0], x["tree"][:0], out[:0])
    fm.tree_attention_fp8(x["q"][:, :0], x["k"][:, :0], x["v"][:, :0], *rest, x["page_table"], x["lengths"], x["tree"][:, :0], out[:, :0])
    none = dict(x, page_table=x["page_table"][:, :0], lengths=torch.zeros_like(x["lengths"]), **{n: x[n][:0] for n in NAMES[3:7]})
    check(run(none), none)                                         # no cache at all
    q = x["q"]
    for at, value in [("q", q.float()), ("q", q.cpu()), ("q", q[..., :96]), ("q", q[:, :, :7]), ("q", q.transpose(2, 3)), ("k", x["k"][:, :2]), ("k", x["k"].bfloat16()),
                      ("v", x["v"][..., :64]), ("v", x["v"].cpu()), ("k_cache", x["k_cache"][:, :, :1]), ("v_cache", x["v_cache"][:1]), ("k_cache", x["k_cache"].cpu()),
                      ("k_cache", _bytes(x["k_cache"])), ("v_cache", x["v_cache"].half()), ("k_scales", x["k_scales"].int()), ("v_scales", x["v_scales"][:, :1]), ("v_scales", x["v_scales"].cpu()),
                      ("k_scales", x["k_scales"].view(torch.int8)), ("k_cache", torch.zeros((*x["k_cache"].shape[:3], 136), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[..., :128]),
                      ("page_table", x["page_table"].long()), ("page_table", x["page_table"][:1]), ("page_table", x["page_table"].t().contiguous().t()), ("lengths", x["lengths"].long()),
                      ("lengths", x["lengths"].cpu()), ("lengths", x["lengths"][:1]), ("tree", x["tree"].int()), ("tree", x["tree"][:, :2]), ("tree", x["tree"].cpu())]:
        with pytest.raises(RuntimeError):
            call(at, value)
    for o in (out.bfloat16(), out[:1], out.cpu(), out.expand(2, 3, 8, 128).transpose(2, 3), out[:1].expand(2, 3, 8, 128)):
        with pytest.raises(RuntimeError):
            call(o=o)
    big = inputs(1, 64, 2, 2, 64, [5], 16)
    with pytest.raises(RuntimeError):
        fm.tree_attention_fp8(*(torch.cat([big[n]] * 2, 1) if n in "qkv" else big[n] for n in NAMES[:-1]), torch.cat([big["tree"]] * 2, 1), torch.cat([big["q"]] * 2, 1).contiguous())
