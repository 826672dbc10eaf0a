"""verify_drafts against the rule of its docstring in 64 bits, token by token; all results are whole numbers and have to be equal.

Probabilities are multiples of 2^-20 or so and their sums lie well apart from the drawn numbers, or differ from them by far more than the 2^-50 by which sums in 64 bits
differ with their order: a case in which two answers lie that near to one another would be a coincidence of 10^-10.
"""
import math

import pytest
import torch

import fp6_marlin_b200 as fm

pytestmark = pytest.mark.gpu


def rule(target, drafted, tree, uniforms, draft=None):
    """On the CPU, with Python's loops: (accepted, counts, next_tokens)."""
    b, t, vocab = target.shape
    accepted, counts, chosen = torch.full((b, t), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32), torch.full((b,), -1)
    clean = lambda x: torch.where((x > 0) & (x < math.inf), x, 0).double()          # noqa: E731
    for s in range(b):
        masks = [int(m) & (1 << 64) - 1 for m in (tree if tree.dim() == 1 else tree[s])]
        if masks[0] == 0:
            continue
        parent = [max((j for j in range(i) if m >> j & 1), default=-1) if m else -2 for i, m in enumerate(masks)]
        way, ids, u = [0], drafted[s].tolist(), uniforms[s].double().tolist()
        r = clean(target[s, 0])
        for i in range(1, t):
            if parent[i] != way[-1]:
                continue
            inside = 0 <= ids[i] < vocab
            if draft is None:
                q = torch.zeros(vocab, dtype=torch.float64)
                if inside:
                    q[ids[i]] = 1
            else:
                q = clean(draft[s, way[-1]])
            if inside and u[i] * float(q[ids[i]]) < float(r[ids[i]]):
                way.append(i)
                r = clean(target[s, i])
                continue
            r = torch.where(q > 0, 0.0, r) if draft is None else (r - q).clamp(min=0)
            r = r / r.sum() if float(r.sum()) > 0 else torch.zeros_like(r)
        if not float(r.sum()) > 0:
            r = clean(target[s, way[-1]])
        up = r.cumsum(0)
        if float(up[-1]) > 0:
            over = (up > u[0] * float(up[-1])).nonzero()
            chosen[s] = int(over[0]) if len(over) else int(r.nonzero()[-1])
        accepted[s, : len(way)], counts[s] = torch.tensor(way, dtype=torch.int32), len(way)
    return accepted, counts, chosen


def trees(b, t, seed, chain=False):
    gen = torch.Generator().manual_seed(seed)
    parents = (torch.rand((b, t), generator=gen) * torch.arange(t)).long() - 1
    parents[:, 1:].clamp_(min=0)
    if chain:
        parents = (torch.arange(t) - 1).expand(b, t)
    return fm.tree_masks(parents), parents


def inputs(b, t, vocab, dtype=torch.float32, with_draft=True, seed=0, chain=False, sharp=3.0):
    gen = torch.Generator().manual_seed(seed + b + 10 * t + vocab)
    logits = sharp * torch.randn((b, t, vocab), generator=gen)
    target = torch.softmax(logits, 2).to(dtype)
    rough = torch.softmax(logits + 0.7 * torch.randn((b, t, vocab), generator=gen), 2)
    tree, parents = trees(b, t, seed, chain)
    drawn = torch.multinomial(rough.view(b * t, vocab), t, replacement=True, generator=gen).view(b, t, t)
    drafted = drawn[torch.arange(b)[:, None], parents.clamp(min=0), torch.arange(t)]
    return {"target": target.cuda(), "drafted": drafted.cuda(), "tree": tree.cuda(), "uniforms": torch.rand((b, t), generator=gen).cuda(), "draft": rough.to(dtype).cuda() if with_draft else None}


def run(x):
    b, t, _ = x["target"].shape
    outs = [torch.full((b, t), 77, dtype=torch.int32, device="cuda"), torch.full((b,), 77, dtype=torch.int32, device="cuda"), torch.full((b,), 77, device="cuda")]
    fm.verify_drafts(x["target"], x["drafted"], x["tree"], x["uniforms"], *outs, draft=x["draft"])
    return outs


def check(x):
    got, want = run(x), rule(*(x[n].cpu() for n in ("target", "drafted", "tree", "uniforms")), None if x["draft"] is None else x["draft"].cpu())
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b.to(a.dtype)), (a, b)
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("b,t,vocab,chain", [(1, 1, 1, True), (1, 1, 7, True), (3, 1, 1000, True), (1, 2, 33, True), (4, 5, 129, False), (2, 16, 5000, False), (7, 8, 4097, True), (1, 64, 511, False),
                                             (33, 3, 257, False), (2, 4, 50257, False), (1, 7, 131072, True), (5, 64, 64, False)])
def test_verify(b, t, vocab, chain, with_draft, dtype):
    for seed in range(3):
        x = inputs(b, t, vocab, dtype, with_draft, seed, chain)
        got = check(x)
        assert all(torch.equal(a, c) for a, c in zip(got, run(x)))


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("b", [18, 19])
def test_long_rows_of_as_many_sequences_as_get_wide_clusters_and_of_one_more(b, with_draft):
    check(inputs(b, 3, 70001, with_draft=with_draft))


@pytest.mark.parametrize("with_draft", [True, False])
def test_many_children_that_are_not_accepted(with_draft):
    """All hang on token 0: r is reduced up to 63 times, some ids come twice, some not from the vocabulary."""
    x = inputs(6, 64, 300, with_draft=with_draft, sharp=1.0)
    x["tree"] = fm.tree_masks(torch.tensor([-1] + [0] * 63)).cuda()
    x["uniforms"][:, 1:] = 0.99999
    x["drafted"][1, 5:9] = x["drafted"][1, 4]
    x["drafted"][2, 3:6] = torch.tensor([-1, 300, 1 << 40], device="cuda")
    x["drafted"][3, 1:] = 7
    x["drafted"][4] = torch.arange(64)
    got = check(x)
    if not with_draft:                                             # (drawn children are accepted where the target gives them more than the draft)
        assert int(got[1].min()) == 1


@pytest.mark.parametrize("accepted", [None, 63, 40])
def test_the_target_gives_drafted_tokens_nothing(accepted):
    """Up to 63 children of token 0 without any probability; the sums are those of r reduced by q again and again."""
    x = inputs(3, 64, 2000, sharp=1.0)
    x["tree"] = fm.tree_masks(torch.tensor([-1] + [0] * 63)).cuda()
    x["drafted"] = torch.stack([torch.randperm(2000, generator=torch.Generator().manual_seed(s))[:64] for s in range(3)]).cuda()
    x["target"][:, 0].scatter_(1, x["drafted"], 0.0)
    x["draft"][:] = x["draft"] * 2.0 ** -8                        # (so that something remains of r)
    if accepted:
        x["target"][:, 0].scatter_(1, x["drafted"][:, accepted:accepted + 1], 0.5)
        x["uniforms"][:, accepted] = 0.25
    got = check(x)
    assert got[1].tolist() == [2 if accepted else 1] * 3


def test_ways_and_their_ends():
    """Everything accepted, nothing accepted, the second child accepted, tokens that no way leads to, padding."""
    b, t, vocab = 6, 6, 50
    x = inputs(b, t, vocab)
    #                            0   1  2  3  4  5
    parents = torch.tensor([[-1, 0, 1, 2, 3, 4], [-1, 0, 0, 1, 2, 4], [-1, 0, 0, 2, 3, 4], [-1, -1, 0, 1, 2, 2], [-2, 0, 0, 0, 0, 0], [-1, 0, 0, -2, 2, 2]])
    parents[4, 1:] = -2
    x["tree"] = fm.tree_masks(parents).cuda()
    for s, n, c, ratio in ((0, 0, 1, 2), (0, 1, 2, 2), (0, 2, 3, 2), (0, 3, 4, 2), (0, 4, 5, 2), (2, 0, 2, 2)):
        x["target"][s, n, x["drafted"][s, c]] = 0.9                # more than the draft gives: accepted
    x["uniforms"][0, 1:] = 0.0
    x["uniforms"][1, 1:] = 0.9999
    x["target"][1, 0, x["drafted"][1, 1]] = x["target"][1, 0, x["drafted"][1, 2]] = 0.0
    x["target"][2, 0, x["drafted"][2, 1]] = 0.0
    accepted, counts, next_tokens = check(x)
    assert accepted[0].tolist() == [0, 1, 2, 3, 4, 5] and counts[1] == 1 and accepted[2, :2].tolist() == [0, 2] and counts[4] == 0 and next_tokens[4] == -1
    x["draft"] = None
    check(x)
    x["tree"] = x["tree"][0].contiguous()                          # one for all
    check(x)


@pytest.mark.parametrize("with_draft", [True, False])
def test_rows_that_hold_nothing_and_values_that_are_no_probabilities(with_draft):
    x = inputs(8, 4, 700, with_draft=with_draft)
    x["target"][0] = 0
    x["target"][1, :, 5:] = float("nan")
    x["target"][2, :, ::2] = -1.0
    x["target"][3, :, 3] = float("inf")
    x["target"][4] = x["draft"][4] if with_draft else x["target"][4]        # nothing remains of r after the first child
    x["target"][5] = 0
    x["target"][5, :, 699] = 2.0 ** -40                            # a single value, the last
    x["uniforms"][4, 1:] = 1.0
    x["uniforms"][6] = torch.tensor([1.0, 0.5, 0.5, 0.5])          # at and beyond the end: the last token that has a probability
    x["uniforms"][7] = float("nan")
    if with_draft:
        x["draft"][2, :, 1::2] = float("nan")
        x["draft"][6] = 0
    got = check(x)
    assert got[2][0] == -1 and got[2][5] == 699


def test_the_first_and_the_last_token_and_borders_between_stretches():
    """Equal probabilities, exact in 64 bits: the next token is known for every drawn number, also where it falls on a sum."""
    vocab = 1 << 14
    at = torch.tensor([0, 1, 31, 127, 128, 511, 512, 513, 4095, 4096, 8191, 8192, vocab - 2, vocab - 1])
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for shift in (0.0, 0.5):                                   # on the border: the token above it
            target = torch.full((len(at), 1, vocab), 1.0 / vocab, dtype=dtype, device="cuda")
            x = {"target": target, "drafted": torch.zeros((len(at), 1), dtype=torch.long, device="cuda"), "tree": torch.ones(1, dtype=torch.long, device="cuda"),
                 "uniforms": ((at + shift) / vocab).float()[:, None].cuda(), "draft": None}
            assert torch.equal(run(x)[2].cpu(), at)


def test_the_tokens_are_distributed_as_the_target_says():
    """Of N independent draws a token's share differs from its probability by a standard deviation of sqrt(p (1 - p) / N); five of them."""
    n, vocab = 40000, 6
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = torch.tensor([0.3, 0.05, 0.25, 0.1, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.05, 0.35, 0.2, 0.2, 0.1, 0.1], device="cuda")
    for draft in (True, False):
        children = torch.multinomial(q.expand(n, vocab), 2, replacement=draft, generator=gen)
        drafted = torch.cat([torch.zeros((n, 1), dtype=torch.long, device="cuda"), children], 1)
        x = {"target": p.expand(n, 3, vocab).contiguous(), "drafted": drafted, "tree": fm.tree_masks(torch.tensor([-1, 0, 0])).cuda(), "uniforms": torch.rand((n, 3), generator=gen, device="cuda"),
             "draft": q.expand(n, 3, vocab).contiguous() if draft else None}
        accepted, counts, next_tokens = run(x)
        first = torch.where(counts > 1, drafted.gather(1, accepted[:, 1:2].clamp(min=0).long())[:, 0], next_tokens)
        share = torch.bincount(first, minlength=vocab).float() / n
        assert ((share - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all(), (share, p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    """Rows that start anywhere, rows among others, target and draft apart by other steps."""
    x = inputs(3, 6, 1003, dtype)
    want = run(x)
    for lead in (1, 3):
        y = dict(x)
        wide = torch.zeros((3, 6, 1003 + 2 * lead), dtype=dtype, device="cuda")
        wide[..., lead:-lead] = x["target"]
        y["target"] = wide[..., lead:-lead]
        assert all(torch.equal(a, b) for a, b in zip(run(y), want))
        y["draft"] = x["draft"].transpose(0, 1).contiguous().transpose(0, 1)
        assert all(torch.equal(a, b) for a, b in zip(run(y), want))
    y = dict(x, target=x["target"][:1].expand(3, 6, 1003), draft=x["draft"][:, :1].expand(3, 6, 1003))
    check(y)
    y["tree"] = torch.cat([x["tree"], x["tree"]], 1)[:, :6]
    check(y)


def test_streams_and_graph():
    sets = [inputs(4, 8, 9000, seed=s) for s in (1, 2)]
    want = [run(x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = run(sets[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got, expect in zip(outs, want) for a, b in zip(got, expect))
    graph, x, got = torch.cuda.CUDAGraph(), sets[0], run(sets[0])
    with torch.cuda.graph(graph, stream=streams[0]):
        fm.verify_drafts(x["target"], x["drafted"], x["tree"], x["uniforms"], *got, draft=x["draft"])
    for other in (inputs(4, 8, 9000, seed=s) for s in (5, 6, 7)):
        for n in ("target", "drafted", "tree", "uniforms", "draft"):
            x[n].copy_(other[n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run(x)))
        check(x)


def test_nothing_to_do_and_refusals():
    x = inputs(2, 3, 100)
    outs = run(x)
    names = ("target", "drafted", "tree", "uniforms", "accepted", "counts", "next_tokens")
    good = dict(zip(names, (x["target"], x["drafted"], x["tree"], x["uniforms"], *outs)), draft=x["draft"])
    fm.verify_drafts(**good)
    fm.verify_drafts(**{n: v[:0] for n, v in good.items()})
    t, d = x["target"], x["drafted"]
    for at, value in [("target", t.double()), ("target", t.cpu()), ("target", t[0]), ("target", t.transpose(1, 2).contiguous().transpose(1, 2)), ("target", t[..., :0]), ("target", t[:, :2]), ("draft", t.half()),
                      ("draft", t[:, :2]), ("draft", t.cpu()), ("draft", t[..., :99]), ("draft", t.transpose(1, 2).contiguous().transpose(1, 2)), ("drafted", d.int()), ("drafted", d[:1]), ("drafted", d.cpu()),
                      ("drafted", d.t().contiguous().t()), ("tree", x["tree"].int()), ("tree", x["tree"][:, :2]), ("tree", x["tree"].t().contiguous().t()), ("tree", x["tree"].cpu()), ("uniforms", x["uniforms"].double()),
                      ("uniforms", x["uniforms"][:1]), ("uniforms", x["uniforms"].cpu()), ("accepted", outs[0].long()), ("accepted", outs[0][:1]), ("accepted", outs[0].cpu()), ("counts", outs[1].long()),
                      ("counts", outs[1][:1]), ("next_tokens", outs[2].int()), ("next_tokens", outs[2].cpu()), ("next_tokens", outs[2][:1])]:
        with pytest.raises(RuntimeError):
            fm.verify_drafts(**dict(good, **{at: value}))
    big = inputs(1, 64, 8)
    with pytest.raises(RuntimeError):
        fm.verify_drafts(torch.cat([big["target"]] * 2, 1), torch.cat([big["drafted"]] * 2, 1), torch.cat([big["tree"]] * 2, 1), torch.cat([big["uniforms"]] * 2, 1),
                         torch.zeros((1, 128), dtype=torch.int32, device="cuda"), outs[1][:1], outs[2][:1])
