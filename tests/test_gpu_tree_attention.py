"""tree_attention against softmax attention in 64 bits.

Bounds, with u = 2^-11 (fp16) or 2^-8 (bf16): the result is rounded once (u of itself) and the weights of the softmax once before they
meet the values (u of sum p |v|, and as much again where their sum is taken of the unrounded ones).  Scores are fp32 sums of D products, each addition
off by at most 2^-23: D * 2^-23 * scale * sum |q k| in the exponent, twice (weight and total), plus 2^-20 for the exponentials and the running sums.
"""
import math

import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu

BITS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _inputs(b, t, h, g, d, lengths, page, dtype=torch.float16, seed=0, spare=2, fill=None):
    gen = torch.Generator(device="cuda").manual_seed(seed + b + 3 * t + 5 * h + 7 * d + 11 * page)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    per = max(1, -(-int(lengths.max()) // page))
    pages = b * per + spare
    qkv = torch.randn((b, t, (h + 2 * g) * d), generator=gen, device="cuda").to(dtype)
    kc, vc = (torch.randn((pages, page, g, d), generator=gen, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: b * per].view(b, per).int().cuda()
    parents = torch.tensor([[(i * 7 + r) % (i + 1) - 1 for i in range(t)] for r in range(b)])
    x = {"q": qkv[..., : h * d].unflatten(2, (h, d)), "k": qkv[..., h * d:(h + g) * d].unflatten(2, (g, d)), "v": qkv[..., (h + g) * d:].unflatten(2, (g, d)),
         "k_cache": kc, "v_cache": vc, "page_table": table, "lengths": lengths.cuda(), "tree": fm.tree_masks(parents).cuda()}
    if fill is not None:          # what must not be read: slots behind the last token, pages of nobody
        used = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
        for i, n in enumerate(lengths.tolist()):
            at = torch.arange(n, device="cuda")
            used[table[i].long()[at // page], at % page] = True
        kc[~used], vc[~used] = fill, fill
    return x


def _exact(x, scale=None):
    q, k, v, tree = x["q"].double(), x["k"].double(), x["v"].double(), x["tree"].cpu()
    b, t, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    page, group = x["k_cache"].shape[1], h // k.shape[2]
    out, size, slack = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((b, t, h, 1), dtype=torch.float64, device="cuda")
    for i, n in enumerate(x["lengths"].tolist()):
        at = torch.arange(n, device="cuda")
        rows, slots = x["page_table"][i].long()[at // page], at % page
        keys = torch.cat([x["k_cache"][rows, slots].double(), k[i]]).repeat_interleave(group, 1)              # n + t, h, d
        values = torch.cat([x["v_cache"][rows, slots].double(), v[i]]).repeat_interleave(group, 1)
        for j in range(t):
            word = int(tree[j] if tree.dim() == 1 else tree[i, j])
            if word == 0:
                continue
            seen = torch.tensor([True] * n + [bool(word >> c & 1) for c in range(t)], device="cuda")
            ks, vs = keys[seen], values[seen]
            s = torch.einsum("hd,nhd->hn", q[i, j], ks) * scale
            p = torch.softmax(s, 1)
            out[i, j] = torch.einsum("hn,nhd->hd", p, vs)
            size[i, j] = torch.einsum("hn,nhd->hd", p, vs.abs())
            slack[i, j] = (torch.einsum("hd,nhd->hn", q[i, j].abs(), ks.abs()) * abs(scale)).amax(1, keepdim=True) * d * 2.0 ** -23
    return out, size, slack


def _run(x, **more):
    out = torch.full(x["q"].shape, float("nan"), dtype=x["q"].dtype, device="cuda")
    fm.tree_attention(*(x[n] for n in ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")), out, **more)
    return out


def _check(out, x, scale=None):
    expect, size, slack = _exact(x, scale)
    u = BITS[out.dtype]
    err, bound = (out.double() - expect).abs(), u * expect.abs() + (2 * u + 2 * slack + 2.0 ** -20) * size + 2.0 ** -25
    assert (err <= bound).all(), float((err / bound).max())


CASES = [
    # b, t, heads, kv heads, d, lengths, page (up to 32 rows of a head of keys, up to 128, more; whole runs of a page and single tokens)
    (1, 1, 1, 1, 128, [0], 16), (1, 1, 32, 32, 128, [1], 16), (1, 1, 32, 32, 128, [300], 16), (1, 1, 8, 1, 64, [63], 16), (1, 1, 8, 1, 64, [64], 16),
    (2, 1, 8, 8, 64, [65, 0], 1), (3, 5, 32, 8, 128, [0, 1000, 17], 16), (1, 64, 64, 8, 128, [500], 48), (2, 64, 8, 8, 64, [129, 2048], 64), (1, 16, 1, 1, 128, [4097], 24),
    (4, 7, 10, 2, 128, [5, 6, 7, 8], 3), (2, 33, 9, 3, 64, [100, 31], 7), (1, 3, 64, 1, 128, [1025], 256), (5, 2, 4, 4, 128, [900, 3, 64, 128, 127], 128),
    (17, 4, 16, 2, 128, list(range(0, 17 * 40, 40)), 16), (1, 1, 64, 8, 128, [20000], 16), (1, 64, 32, 4, 128, [9000], 16), (70, 1, 8, 2, 64, [i * 5 for i in range(70)], 32),
    (1, 17, 8, 8, 128, [777], 4096), (3, 64, 3, 1, 128, [64, 0, 200], 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,g,d,lengths,page", CASES)
def test_attention(b, t, h, g, d, lengths, page, dtype):
    x = _inputs(b, t, h, g, d, lengths, page, dtype, fill=float("nan"))
    for _ in range(2):
        out = _run(x)
        _check(out, x)
    assert torch.equal(out, _run(x)) and fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", [(1, 4, 1, 128), (8, 32, 4, 128), (7, 8, 1, 64), (16, 8, 1, 128), (40, 8, 2, 64)])
def test_rows_joined_from_many_ranges(t, h, g, d):
    """One long sequence and few heads of keys: every multiprocessor leaves a part of the same rows; few and many rows after one another."""
    x, other = _inputs(1, t, h, g, d, [12345], 16, torch.bfloat16), _inputs(1, 3, 2, 1, d, [4321], 16, torch.bfloat16)
    first, first_other = _run(x), _run(other)
    _check(first, x)
    _check(first_other, other)
    for _ in range(5):
        assert torch.equal(_run(x), first) and torch.equal(_run(other), first_other)
    x["v"][0, 0, 0, 3] = float("inf")                                # it reaches the rows that see it through the joined parts as well
    heads = h // g
    out, sees = _run(x)[0].float(), (x["tree"].reshape(-1) & 1).bool()
    assert (out[:, :heads, 3].isposinf() == sees[:, None]).all() and out[~sees].isfinite().all() and fm.device_status() == 0


@pytest.mark.parametrize("lengths", [[0, 0], [200, 0], [65, 1300]])
def test_padding_and_rows_that_see_nothing(lengths):
    x = _inputs(2, 6, 8, 2, 128, lengths, 16, fill=float("inf"))
    x["tree"][0, 2] = 0
    x["tree"][1, 3:] = 0
    x["tree"][1, 0] = 0b000010                                     # sees another token, not itself
    x["k"][0, 2], x["v"][0, 2] = float("nan"), float("nan")        # what padding holds is seen by nobody
    x["k"][1, 3:], x["v"][1, 3:] = float("inf"), float("-inf")
    x["tree"] &= ~torch.tensor([[0b100], [0b111000]], device="cuda")
    out = _run(x)
    assert (out[0, 2] == 0).all() and (out[1, 3:] == 0).all()
    clean = {n: v.clone() for n, v in x.items()}
    for n in ("k", "v"):
        clean[n][0, 2], clean[n][1, 3:] = 0, 0
    _check(out, clean)


@pytest.mark.parametrize("length", [0, 40, 700])
def test_values_that_are_not_finite_reach_those_that_see_them(length):
    """Token 1 sees token 0 and itself, token 2 only itself; token 0's values hold an infinity and a NaN."""
    x = _inputs(1, 3, 4, 2, 64, [length], 16)
    x["tree"] = torch.tensor([0b001, 0b011, 0b100], device="cuda")
    x["v"][0, 0, 0, 5], x["v"][0, 0, 1, 7] = float("inf"), float("nan")
    out = _run(x).float()
    assert out[0, :2, :2, 5].isposinf().all() and out[0, :2, 2:, 7].isnan().all()
    assert out[0, 2].isfinite().all()
    clean = {n: v.clone() for n, v in x.items()}
    clean["v"][0, 0, 0, 5], clean["v"][0, 0, 1, 7] = 0, 0
    rest = _run(clean)
    out[0, :2, :2, 5], out[0, :2, 2:, 7] = rest[0, :2, :2, 5].float(), rest[0, :2, 2:, 7].float()
    _check(out.to(rest.dtype), clean)


@pytest.mark.parametrize("t", [1, 20])
def test_large_scores_and_scale(t):
    """Scores in the thousands: the running maximum keeps every exponential in range."""
    x = _inputs(2, t, 8, 2, 128, [300, 70], 16)
    x["q"] = x["q"] * 30
    x["k_cache"] *= 30
    _check(_run(x, scale=1.0), x, 1.0)
    _check(_run(x, scale=-0.5), x, -0.5)
    zero = _run(x, scale=0.0)                                      # the mean of what is seen
    _check(zero, x, 0.0)


def test_one_mask_for_all_and_strided_tensors():
    x = _inputs(3, 4, 8, 4, 128, [50, 0, 333], 16)
    chain = fm.tree_masks(torch.arange(4) - 1).cuda()
    x["tree"] = chain
    one = _run(x)
    _check(one, x)
    # heads first, the cache's heads before its slots, a page table and masks with longer rows
    y = dict(x)
    y["q"] = x["q"].transpose(1, 2).contiguous().transpose(1, 2)
    y["k_cache"] = x["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    y["v_cache"] = torch.cat([x["v_cache"], x["v_cache"]], 3)[..., :128]
    y["page_table"] = torch.cat([x["page_table"], torch.full((3, 2), 1 << 30, dtype=torch.int32, device="cuda")], 1)[:, : x["page_table"].shape[1]]
    y["tree"] = torch.cat([chain.expand(3, 4), torch.zeros((3, 1), dtype=torch.int64, device="cuda")], 1)[:, :4]
    out = torch.zeros((3, 8, 4, 128), dtype=torch.float16, device="cuda").transpose(1, 2)
    fm.tree_attention(*(y[n] for n in ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")), out)
    assert torch.equal(out, one)


def test_strides_of_single_places():
    """One sequence, one token, one head of keys, one page: whatever their strides are."""
    x = _inputs(1, 1, 4, 1, 64, [9], 16, spare=0)
    expect = _run(x)
    for n, at in (("k", (0, 1, 2)), ("v", (0, 1, 2)), ("k_cache", (0, 2)), ("v_cache", (0, 2)), ("q", (0, 1))):
        steps = [1 if i in at else s for i, s in enumerate(x[n].stride())]
        x[n] = x[n].contiguous().as_strided(x[n].shape, steps)
    assert torch.equal(_run(x), expect)


def test_lengths_and_pages_out_of_range():
    x = _inputs(3, 2, 4, 2, 128, [64, 48, 80], 16)
    same = {n: v.clone() for n, v in x.items()}
    x["lengths"] = torch.tensor([1 << 30, -5, 80], dtype=torch.int32, device="cuda")      # cut to the table, to zero
    same["lengths"] = torch.tensor([80, 0, 80], dtype=torch.int32, device="cuda")
    x["page_table"][0, 4] = same["page_table"][0, 4] = same["page_table"][0, 3]
    assert torch.equal(_run(x), _run(same)) and fm.device_status() == 0
    x["lengths"] = same["lengths"] = torch.tensor([64, 48, 80], dtype=torch.int32, device="cuda")
    for wrong in (-1, x["k_cache"].shape[0], 1 << 30):
        x["page_table"][2, 4] = wrong                              # the last page: hidden, as if the sequence were shorter
        out = _run(x)
        assert fm.device_status() == 4
        same["lengths"] = torch.tensor([64, 48, 64], dtype=torch.int32, device="cuda")
        expect, size, slack = _exact(same)
        u = BITS[out.dtype]
        assert ((out.double() - expect).abs() <= u * expect.abs() + (2 * u + 2 * slack + 2.0 ** -20) * size + 2.0 ** -25).all()


def test_long_cache_offsets():
    """A cache of more than 2^31 values, whose last pages are used."""
    g, d, page = 8, 128, 128
    pages = (1 << 31) // (page * g * d) + 9
    kc = torch.zeros((pages, page, g, d), dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    x = _inputs(1, 2, 16, g, d, [1000], page)
    table = torch.arange(pages - 8, pages, device="cuda").flip(0)[None].int()
    kc[table[0].long()], vc[table[0].long()] = x["k_cache"][x["page_table"][0].long()], x["v_cache"][x["page_table"][0].long()]
    expect = _run(x)
    x["k_cache"], x["v_cache"], x["page_table"] = kc, vc, table
    assert torch.equal(_run(x), expect)


def test_streams_and_graph():
    sets = [_inputs(2, 5, 32, 8, 128, [3000, 1000 + seed], 16, seed=seed) for seed in (1, 2)]
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
    call = lambda: fm.tree_attention(*(x[n] for n in ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")), out)     # noqa: E731
    with torch.cuda.graph(graph, stream=streams[0]):
        call()
    for n in (3000, 7, 0):                                         # lengths are the device's: one graph serves all
        x["lengths"][0] = n
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x)


def test_nothing_to_do_and_refusals():
    x = _inputs(2, 3, 8, 2, 128, [20, 30], 16)
    names = ("q", "k", "v", "k_cache", "v_cache", "page_table", "lengths", "tree")
    good = [x[n] for n in names]
    out = torch.empty_like(x["q"].contiguous())

    def call(at=None, value=None, o=out):
        args = list(good)
        if at is not None:
            args[names.index(at)] = value
        fm.tree_attention(*args, o)

    call()
    fm.tree_attention(x["q"][:0], x["k"][:0], x["v"][:0], x["k_cache"], x["v_cache"], x["page_table"][:0], x["lengths"][:0], x["tree"][:0], out[:0])
    fm.tree_attention(x["q"][:, :0], x["k"][:, :0], x["v"][:, :0], x["k_cache"], x["v_cache"], x["page_table"], x["lengths"], x["tree"][:, :0], out[:, :0])
    none = dict(x, k_cache=x["k_cache"][:0], v_cache=x["v_cache"][:0], page_table=x["page_table"][:, :0], lengths=torch.zeros_like(x["lengths"]))
    _check(_run(none), none)                                       # no cache at all
    q = x["q"]
    for at, value in [("q", q.float()), ("q", q.cpu()), ("q", q[..., :96]), ("q", q[:, :, :7]), ("q", q.transpose(2, 3)), ("k", x["k"][:, :2]), ("k", x["k"].bfloat16()),
                      ("v", x["v"][..., :64]), ("v", x["v"].cpu()), ("k_cache", x["k_cache"][:, :, :1]), ("v_cache", x["v_cache"][:1]), ("k_cache", x["k_cache"].cpu()),
                      ("page_table", x["page_table"].long()), ("page_table", x["page_table"][:1]), ("page_table", x["page_table"].t().contiguous().t()), ("lengths", x["lengths"].long()),
                      ("lengths", x["lengths"].cpu()), ("lengths", x["lengths"][:1]), ("tree", x["tree"].int()), ("tree", x["tree"][:, :2]), ("tree", x["tree"].cpu())]:
        with pytest.raises(RuntimeError):
            call(at, value)
    for o in (out.bfloat16(), out[:1], out.cpu(), out.expand(2, 3, 8, 128).transpose(2, 3), out[:1].expand(2, 3, 8, 128)):
        with pytest.raises(RuntimeError):
            call(o=o)
    big = _inputs(1, 64, 2, 2, 64, [5], 16)
    with pytest.raises(RuntimeError):
        fm.tree_attention(*(torch.cat([big[n]] * 2, 1) if n in "qkv" else big[n] for n in names[:-1]), torch.cat([big["tree"]] * 2, 1), torch.cat([big["q"]] * 2, 1).contiguous())


@pytest.mark.parametrize("t,h,g,d", [(1, 4, 1, 128), (3, 8, 2, 64), (5, 8, 1, 128), (40, 16, 2, 128), (63, 2, 1, 64)])
def test_bits_behind_the_last_token(t, h, g, d):
    """They stand for no token; an entry that has only such bits is not 0, so not padding: it sees the committed tokens."""
    x = _inputs(3, t, h, g, d, [200, 64, 7], 16)
    expect = _run(x)
    x["tree"] |= -1 << t
    assert torch.equal(_run(x), expect)
    x["tree"][:, t // 2] = 1 << t if t < 63 else -(1 << 63)
    x["tree"][2, 0] = -(1 << 63)
    x["tree"][1, t - 1] = 0
    _check(_run(x), x)


def test_tables_and_masks_of_single_places():
    """One page a sequence, one drafted token, one sequence: the step to a next one that there is not may be anything."""
    x = _inputs(3, 1, 4, 1, 64, [9, 16, 0], 16)
    expect = _run(x)
    x["page_table"], x["tree"] = x["page_table"].t().contiguous().t(), x["tree"].t().contiguous().t()
    for n in ("page_table", "tree"):
        x[n] = x[n].as_strided((3, 1), (1, 3))
    assert torch.equal(_run(x), expect)
    one = _inputs(1, 1, 4, 1, 64, [9], 16)
    expect = _run(one)
    one["lengths"], one["tree"] = one["lengths"].as_strided((1,), (5,)), one["tree"][0].as_strided((1,), (7,))
    one["page_table"] = one["page_table"].as_strided((1, 1), (4, 6))
    assert torch.equal(_run(one), expect)
