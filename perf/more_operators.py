"""The operators around an 8-bit cache and the choice among drafted tokens, as cases that can be timed.

Keys and values written into a paged cache in E4M3 with a power of two for each token and head, read back from it, attention of drafted
or single tokens over it, and the verification of drafted tokens against the target's probabilities from given random numbers.  With ``own``
the calls are those of ``fp6_marlin_b200``; without it the same formulas in elementary torch operations in 32 bits (64 for the probabilities).
"""
import math

import torch

own = False

E4M3_MAX = 448.0
# exponents of the powers of two, and the largest E4M3 value at the highest of them: what is read back is finite in the type that was written
RANGES = {torch.float16: (-15, 8), torch.bfloat16: (-40, 120)}
AT_THE_TOP = 240.0

MOST_WRITTEN = 4 * 4096 * 8       # tokens x heads of keys
MOST_READ = 16 * 6144 * 8
MOST_KV_TOKENS = 64 * 8 * 8192    # tokens of the cache x heads of keys and values
MOST_SCORES = 2 * 64 * 64 * 32768 # query heads x drafted tokens x keys
MOST_PROBABILITIES = 64 * 7 * 131072


def listed():
    return [
        # the accepted ones of seven drafted tokens of a few sequences, after a step of verification: latency
        {"name": "write b16 t7 32 l1000 accepted", "kind": "write", "b": 16, "t": 7, "kv": 32, "d": 128, "cache": 1000, "page": 16, "type": "f16", "take": True},
        # the prompts of four sequences at once
        {"name": "write b4 t4096 8 l0", "kind": "write", "b": 4, "t": 4096, "kv": 8, "d": 128, "cache": 0, "page": 64, "type": "bf16", "take": False},
        # a short prefix, read back for one sequence
        {"name": "read b1 32 l300", "kind": "read", "b": 1, "kv": 32, "d": 128, "cache": 300, "page": 16, "type": "f16", "even": True, "part": False},
        # ragged caches of a batch, for a step that needs them in 16 bits
        {"name": "read b16 8 l6144", "kind": "read", "b": 16, "kv": 8, "d": 128, "cache": 6144, "page": 48, "type": "bf16", "even": False, "part": False},
        # the next token of one short sequence, a head of keys for each head of queries: latency
        {"name": "attend b1 t1 32/32 l300", "kind": "attend", "b": 1, "t": 1, "heads": 32, "kv": 32, "d": 128, "cache": 300, "page": 16, "type": "f16", "even": True},
        # the next token of each sequence of a serving batch
        {"name": "attend b64 t1 64/8 l8192", "kind": "attend", "b": 64, "t": 1, "heads": 64, "kv": 8, "d": 128, "cache": 8192, "page": 64, "type": "bf16", "even": False},
        # the next token of a few long documents
        {"name": "attend b3 t1 32/4 l65537", "kind": "attend", "b": 3, "t": 1, "heads": 32, "kv": 4, "d": 128, "cache": 65537, "page": 16, "type": "f16", "even": True},
        # small trees over the ragged caches of a few sequences
        {"name": "attend b8 t5 32/32 l4096", "kind": "attend", "b": 8, "t": 5, "heads": 32, "kv": 32, "d": 128, "cache": 4096, "page": 64, "type": "f16", "even": False},
        # a large tree over two long caches, eight heads of queries to each head of keys: 512 rows share a key
        {"name": "attend b2 t64 64/8 l32768", "kind": "attend", "b": 2, "t": 64, "heads": 64, "kv": 8, "d": 128, "cache": 32768, "page": 16, "type": "bf16", "even": True},
        # nothing drafted beside the last token: a token drawn from one row of probabilities
        {"name": "verify b1 t1 v32000", "kind": "verify", "b": 1, "t": 1, "vocab": 32000, "type": "f32", "draft": False, "chain": True},
        # trees of a few sequences, drafted by a model whose probabilities are kept, a vocabulary of odd size
        {"name": "verify b5 t16 v50257 draft", "kind": "verify", "b": 5, "t": 16, "vocab": 50257, "type": "bf16", "draft": True, "chain": False},
        # a serving batch, a chain of six drafted tokens behind the last one each, a large vocabulary
        {"name": "verify b64 t7 v131072 draft", "kind": "verify", "b": 64, "t": 7, "vocab": 131072, "type": "f32", "draft": True, "chain": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    pick, kind_of, d = rng.random(), rng.choice(["f16", "bf16"]), rng.choice([64, 128, 128])
    page, kv = rng.choice([1, 16, 16, 24, 32, 64, 128, 256]), rng.choice([1, 2, 4, 8, 16, 32])
    if pick < 0.2:
        while True:
            b, take = _log_int(rng, 1, 64), rng.random() < 0.5
            t, cache = _log_int(rng, 1, 64 if take else 4096), _log_int(rng, 1, 4096)
            if b * t * kv <= MOST_WRITTEN and b * kv * cache <= 64 * 8 * 2048:
                return {"kind": "write", "b": b, "t": t, "kv": kv, "d": d, "cache": cache, "page": page, "type": kind_of, "take": take}
    if pick < 0.35:
        while True:
            b, cache = _log_int(rng, 1, 64), _log_int(rng, 16, 32768)
            if b * kv * cache <= MOST_READ:
                return {"kind": "read", "b": b, "kv": kv, "d": d, "cache": cache, "page": page, "type": kind_of, "even": rng.random() < 0.3, "part": rng.random() < 0.5}
    if pick < 0.7:
        while True:
            b, t, cache, group = _log_int(rng, 1, 64), rng.choice([1, 1, _log_int(rng, 1, 64)]), _log_int(rng, 16, 65536), rng.choice([1, 1, 2, 3, 4, 5, 8])
            if b * kv * cache <= MOST_KV_TOKENS and b * t * kv * group * (cache + t) <= MOST_SCORES and kv * group <= 64:
                return {"kind": "attend", "b": b, "t": t, "heads": kv * group, "kv": kv, "d": d, "cache": cache, "page": page, "type": kind_of, "even": rng.random() < 0.3}
    while True:
        b, t, vocab = _log_int(rng, 1, 64), _log_int(rng, 1, 64), _log_int(rng, 1000, 200000)
        if b * t * vocab <= MOST_PROBABILITIES:
            return {"kind": "verify", "b": b, "t": t, "vocab": vocab, "type": rng.choice(["f32", "f32", "f16", "bf16"]), "draft": rng.random() < 0.6, "chain": rng.random() < 0.5}


def _lengths(case):
    """Committed tokens of each sequence: all alike, or ragged from an empty cache to the longest."""
    b, longest = case["b"], case["cache"]
    if case.get("even") or b == 1:
        return [longest] * b
    return [longest * i // (b - 1) for i in range(b)]


def _type(case):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[case["type"]]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _quantised(x):
    """x (..., d) -> E4M3 values and the exponents (plus 127) of their powers of two: the lowest with which the largest magnitude stays within 448."""
    lowest, highest = RANGES[x.dtype]
    top = torch.where(x.isfinite(), x.float().abs(), 0).amax(-1)
    part, power = torch.frexp(top)                                     # top = part * 2 ** power, 448 = 0.875 * 2 ** 9
    power = torch.where(top == 0, lowest, power - torch.where(part > 0.875, 8, 9)).clamp(lowest, highest)
    y = torch.ldexp(x.float(), -power[..., None])
    limit = torch.where(power == highest, AT_THE_TOP, E4M3_MAX)[..., None]
    y = torch.where(x.isfinite(), torch.minimum(torch.maximum(y, -limit), limit), math.nan)
    return y.to(torch.float8_e4m3fn), (power + 127).to(torch.uint8)


def _power(exponents, dtype=torch.float32):
    return (exponents.int() << 23).view(torch.float32).to(dtype)


def _cache(gen, case, pages, dtype):
    """A paged cache that earlier steps have filled: tokens and heads of unlike size."""
    kv, d, page, out = case["kv"], case["d"], case["page"], {}
    for name in ("k", "v"):
        # exponents lie page by page, head by head
        out[name + "_cache"] = torch.empty((pages, page, kv, d), dtype=torch.float8_e4m3fn, device="cuda")
        out[name + "_scales"] = torch.empty((pages, kv, page), dtype=torch.uint8, device="cuda").transpose(1, 2)
        part = max(1, (1 << 26) // (page * kv * d))
        for at in range(0, pages, part):
            here = min(part, pages - at)
            x = torch.randn((here, page, kv, d), generator=gen, device="cuda") * torch.exp(0.5 * _randn(gen, here, page, kv, 1))
            q, e = _quantised(x.to(dtype))
            out[name + "_cache"][at:at + here].copy_(q)
            out[name + "_scales"][at:at + here].copy_(e)
    return out


def _trees(gen, b, t, chain=False, rooted=False):
    """Masks of random trees: the first token hangs on the last committed one, every other on an earlier drafted token (or beside the first)."""
    parent = (torch.rand((b, t), generator=gen) * torch.arange(t)).long() - 1
    parent = torch.where(torch.rand((b, t), generator=gen) < (1.1 if chain else 0.5), torch.arange(t).expand(b, t) - 1, parent)
    if rooted:
        parent[:, 1:].clamp_(min=0)
    see = torch.zeros((b, t, t), dtype=torch.bool)
    for i in range(t):
        p = parent[:, i]
        see[:, i] = torch.where((p >= 0)[:, None], see[torch.arange(b), p.clamp(min=0)], False)
        see[:, i, i] = True
    if b > 2 and t > 2:
        see[1, t - 1] = False     # a sequence with one token fewer: its last place is padding
        see[1, :, t - 1] = False
        parent[1, t - 1] = -2
    return (see.long() << torch.arange(t)).sum(2).cuda(), parent


def _prepare_verify(gen, host, case):
    b, t, vocab, dtype = case["b"], case["t"], case["vocab"], _type(case)
    tree, parent = _trees(host, b, t, case["chain"], True)
    target = torch.empty((b, t, vocab), dtype=dtype, device="cuda")
    draft = torch.empty_like(target) if case["draft"] else None
    proposal = torch.empty((b, t, max(t, 1)), dtype=torch.long, device="cuda")
    for i in range(t):            # a row of logits with a long tail; the drafting model knows them roughly
        logits = 4 * _randn(gen, b, vocab)
        target[:, i] = torch.softmax(logits, 1).to(dtype)
        rough = torch.softmax(logits + 0.8 * _randn(gen, b, vocab), 1)
        if draft is not None:
            draft[:, i] = rough.to(dtype)
        proposal[:, i] = torch.multinomial(rough, max(t, 1), replacement=True, generator=gen)
    at = torch.arange(b)[:, None]
    # a token is one of those that were drawn behind its parent
    drafted = proposal.cpu()[at, parent.clamp(min=0), torch.arange(t)[None, :]].cuda()
    uniforms = torch.rand((b, t), generator=gen, device="cuda")
    return {"target": target, "draft": draft, "drafted": drafted.contiguous(), "tree": tree, "uniforms": uniforms,
            "accepted": torch.empty((b, t), dtype=torch.int32, device="cuda"), "counts": torch.empty(b, dtype=torch.int32, device="cuda"),
            "next": torch.empty(b, dtype=torch.long, device="cuda")}


def prepare(case, seed):
    gen, host, kind, dtype = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed), case["kind"], _type(case)
    if kind == "verify":
        return {"kind": kind, **_prepare_verify(gen, host, case)}
    b, kv, d, page = (case[x] for x in ("b", "kv", "d", "page"))
    t = case.get("t", 0)
    lengths = torch.tensor(_lengths(case))[torch.randperm(b, generator=host)]
    per = -(-max(case["cache"] + (t if kind == "write" else 0), 1) // page)
    pages = b * per
    state = {"kind": kind, **_cache(gen, case, pages, dtype), "pages": torch.randperm(pages, generator=host).view(b, per).int().cuda(), "lengths": lengths.int().cuda()}
    if kind == "read":
        # all of every cache, or a stretch from some token on
        rows = max(1, case["cache"] // 2) if case["part"] else case["cache"]
        state["starts"] = (torch.rand(b, generator=host) * (lengths + 1)).int().cuda() if case["part"] else None
        state["k_out"], state["v_out"] = (torch.zeros((b, rows, kv, d), dtype=dtype, device="cuda") for _ in range(2))
        return state
    # the projection's output: queries, keys and values of a token next to one another
    h = case.get("heads", kv)
    qkv = _randn(gen, b, t, (h + 2 * kv) * d)
    qkv[..., :h * d] *= 2
    qkv = qkv.to(dtype)
    state["k"], state["v"] = qkv[..., h * d:(h + kv) * d].unflatten(2, (kv, d)), qkv[..., (h + kv) * d:].unflatten(2, (kv, d))
    if kind == "write":
        state["tokens"] = state["counts"] = None
        if case["take"]:          # a way through a tree: some of the drafted tokens in order
            counts = 1 + (torch.rand(b, generator=host) * t).long().clamp(max=t - 1)
            picked = (torch.rand((b, t), generator=host) + (torch.arange(t) == 0)).argsort(1, descending=True)
            picked = torch.where(torch.arange(t) < counts[:, None], picked, t).sort(1).values
            state["tokens"], state["counts"] = torch.where(picked == t, -1, picked).int().cuda(), counts.int().cuda()
        return state
    state["q"], state["tree"] = qkv[..., :h * d].unflatten(2, (h, d)), _trees(host, b, t)[0]
    state["out"] = torch.empty((b, t, h, d), dtype=dtype, device="cuda")
    return state


def _run_own(state):
    import fp6_marlin_b200 as fm
    kind = state["kind"]
    if kind == "verify":
        fm.verify_drafts(state["target"], state["drafted"], state["tree"], state["uniforms"], state["accepted"], state["counts"], state["next"], draft=state["draft"])
        return [state["accepted"], state["counts"], state["next"]]
    cache = [state[x] for x in ("k_cache", "v_cache", "k_scales", "v_scales")]
    if kind == "write":
        fm.write_cache_fp8(state["k"], state["v"], *cache, state["pages"], state["lengths"], tokens=state["tokens"], counts=state["counts"])
        return cache
    if kind == "read":
        fm.read_cache_fp8(*cache, state["pages"], state["lengths"], state["k_out"], state["v_out"], starts=state["starts"])
        return [state["k_out"], state["v_out"]]
    fm.tree_attention_fp8(state["q"], state["k"], state["v"], *cache, state["pages"], state["lengths"], state["tree"], state["out"])
    return state["out"]


def _rows_of(tensor, page, slot):
    """Tokens of a cache (E4M3 as bytes: not every indexing operation knows the type)."""
    return tensor.view(torch.uint8)[page, slot].view(tensor.dtype) if tensor.dtype == torch.float8_e4m3fn else tensor[page, slot]


def _write(state):
    b, t = state["k"].shape[:2]
    page_size, device = state["k_cache"].shape[1], state["k"].device
    token = torch.arange(t, device=device).expand(b, t) if state["tokens"] is None else state["tokens"].long()
    entry = torch.arange(t, device=device).expand(b, t)
    if state["counts"] is not None:
        # an entry behind the last writes what the first one does
        entry = torch.where(entry < state["counts"][:, None], entry, 0)
        token = token.gather(1, entry)
    at = state["lengths"].long()[:, None] + entry
    page, slot = state["pages"].long().gather(1, at // page_size), at % page_size
    of = torch.arange(b, device=device)[:, None]
    for name in ("k", "v"):
        q, e = _quantised(state[name][of, token])
        state[name + "_cache"].view(torch.uint8)[page, slot] = q.view(torch.uint8)
        state[name + "_scales"][page, slot] = e
    return [state[x] for x in ("k_cache", "v_cache", "k_scales", "v_scales")]


def _read(state):
    rows, page_size = state["k_out"].shape[1], state["k_cache"].shape[1]
    at = torch.arange(rows, device=state["k_out"].device).expand(state["k_out"].shape[0], rows)
    if state["starts"] is not None:
        at = at + state["starts"].long()[:, None]
    there = at < state["lengths"][:, None]
    at = torch.where(there, at, 0)
    page, slot = state["pages"].long().gather(1, at // page_size), at % page_size
    out = []
    for name in ("k", "v"):
        values = _rows_of(state[name + "_cache"], page, slot).float() * _power(state[name + "_scales"][page, slot])[..., None]
        out.append(torch.where(there[:, :, None, None], values.to(state["k_out"].dtype), state[name + "_out"]))
    return out


def _attend(state):
    q, k, tree, lengths, pages = state["q"], state["k"], state["tree"], state["lengths"], state["pages"].long()
    b, t, h, d = q.shape
    kv, longest = k.shape[2], pages.shape[1] * state["k_cache"].shape[1]
    cached = torch.arange(longest, device=q.device) < lengths[:, None]                                                  # b, longest
    sees = (tree[:, :, None] >> torch.arange(t, device=q.device)) & 1 != 0                                              # b, t, t
    visible = torch.cat([(cached[:, None, :] & (tree != 0)[:, :, None]), sees], 2)                                       # b, t, longest + t

    def tokens(name):
        values = _rows_of(state[name + "_cache"], pages, slice(None)).view(b, longest, kv, d).float()
        values = values * _power(state[name + "_scales"][pages].reshape(b, longest, kv))[..., None]
        return torch.cat([values.masked_fill_(~cached[:, :, None, None], 0), state[name].float()], 1)

    rows = q.float().view(b, t, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, t * (h // kv), d)
    scores = (rows @ tokens("k").permute(0, 2, 3, 1)).view(b, kv, t, h // kv, -1) / math.sqrt(d)
    scores = scores.masked_fill_(~visible[:, None, :, None, :], -math.inf)
    top = scores.amax(4, keepdim=True).clamp(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(4, keepdim=True)
    out = (p.view(b, kv, t * (h // kv), -1) @ tokens("v").transpose(1, 2)).view(b, kv, t, h // kv, d) / total.clamp(min=1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, h, d).to(q.dtype)


def _parents(tree):
    """The last earlier token that each token sees, -1 where there is none."""
    places = torch.arange(tree.shape[-1], device=tree.device)
    earlier = ((tree[..., None] >> places) & 1 != 0) & (places < places[:, None])
    return torch.where(earlier, places + 1, 0).amax(-1) - 1


def _clean(x):
    return torch.where((x > 0) & (x < math.inf), x, 0).double()


def _verify(state):
    target, drafted, tree, uniforms, draft = (state[x] for x in ("target", "drafted", "tree", "uniforms", "draft"))
    b, t, vocab = target.shape
    at, parent = torch.arange(b, device=target.device), _parents(tree)
    alive, node = tree[:, 0] != 0, torch.zeros(b, dtype=torch.long, device=target.device)
    rest = _clean(target[:, 0])                                      # what the next token is drawn from so far
    taken = alive[:, None] & (torch.arange(t, device=target.device) == 0)
    for i in range(1, t):
        child = alive & (tree[:, i] != 0) & (parent[:, i] == node)
        token = drafted[:, i, None].clamp(0, vocab - 1)
        inside = (drafted[:, i] >= 0) & (drafted[:, i] < vocab)
        p = torch.where(inside, rest.gather(1, token)[:, 0], 0)
        if draft is None:
            accept = uniforms[:, i].double() < p
            less = rest.scatter(1, token, torch.where(inside, 0, rest.gather(1, token)[:, 0])[:, None])
        else:
            row = _clean(draft[at, node])
            accept = uniforms[:, i].double() * torch.where(inside, row.gather(1, token)[:, 0], 0) < p
            less = (rest - row).clamp(min=0)
        total = less.sum(1, keepdim=True)
        less = torch.where(total > 0, less / total, 0)
        accept &= child
        rest = torch.where(accept[:, None], _clean(target[:, i]), torch.where(child[:, None], less, rest))
        node = torch.where(accept, i, node)
        taken[:, i] = accept
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, _clean(target[at, node]))
    below = rest.cumsum(1)
    over = below > uniforms[:, :1].double() * below[:, -1:]
    last = torch.where(rest > 0, torch.arange(vocab, device=target.device), -1).amax(1)
    chosen = torch.where(over[:, -1], over.int().argmax(1), last)
    places = torch.arange(t, device=target.device)
    path = torch.where(taken, places, t).sort(1).values
    return [torch.where(path == t, -1, path).int(), taken.sum(1).int(), torch.where(alive, chosen, -1)]


def run(state):
    if own:
        return _run_own(state)
    return {"write": _write, "read": _read, "attend": _attend, "verify": _verify}[state["kind"]](state)


def _exact_quantised(x):
    """Before the rounding to eight bits."""
    lowest, highest = RANGES[x.dtype]
    x = x.double()
    top = x.abs().amax(-1).clamp(min=2.0 ** -140)
    e = torch.ceil(torch.log2(top / 448)).long()
    e += (top > 448 * torch.pow(2.0, e.double())).long() - (top <= 448 * torch.pow(2.0, (e - 1).double())).long()
    e = e.clamp(lowest, highest)
    return x / torch.pow(2.0, e.double())[..., None], (e + 127).to(torch.uint8)


def _exact_verify(state):
    target, draft, b, t = state["target"], state["draft"], *state["target"].shape[:2]
    path, counts, chosen = torch.full((b, t), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32), torch.full((b,), -1)
    for s in range(b):
        masks, ids, u = state["tree"][s].tolist(), state["drafted"][s].tolist(), state["uniforms"][s].double().tolist()
        if masks[0] == 0:
            continue
        way = [0]
        while True:
            here = way[-1]
            p = target[s, here].double()
            left, moved = p, False
            for i in range(here + 1, t):
                earlier = [j for j in range(i) if masks[i] >> j & 1]
                if masks[i] == 0 or not earlier or earlier[-1] != here:
                    continue
                if draft is None:
                    q = torch.zeros_like(p)
                    q[ids[i]] = 1
                else:
                    q = draft[s, here].double()
                if u[i] * float(q[ids[i]]) < float(left[ids[i]]):
                    way.append(i)
                    moved = True
                    break
                left = torch.relu(left - q) if draft is not None else left * (1 - q)
                left = left / left.sum() if float(left.sum()) > 0 else left
            if not moved:
                break
        if float(left.sum()) == 0:
            left = p
        up = torch.cumsum(left, 0)
        chosen[s] = min(int(torch.searchsorted(up, u[0] * up[-1], right=True)), int(left.nonzero()[-1]))
        path[s, :len(way)], counts[s] = torch.tensor(way, dtype=torch.int32), len(way)
    return [path.cuda(), counts.cuda(), chosen.cuda()]


def exact(case, seed):
    state = prepare(case, seed)
    kind, lengths = state["kind"], state["lengths"].tolist() if "lengths" in state else None
    if kind == "verify":
        return _exact_verify(state)
    page, table = state["k_cache"].shape[1], state["pages"].long()

    def place(s, where):
        return table[s][where // page], where % page

    def token_values(name, s, where):
        rows, slots = place(s, where)
        e = state[name + "_scales"][rows, slots].double() - 127
        return _rows_of(state[name + "_cache"], rows, slots).double() * torch.pow(2.0, e)[..., None]

    if kind == "write":
        out = {}
        for name in ("k", "v"):
            values, powers = state[name + "_cache"].double(), state[name + "_scales"].clone()
            for s, n in enumerate(lengths):
                count = state["k"].shape[1] if state["counts"] is None else int(state["counts"][s])
                which = torch.arange(count, device="cuda") if state["tokens"] is None else state["tokens"][s, :count].long()
                rows, slots = place(s, n + torch.arange(count, device="cuda"))
                values[rows, slots], powers[rows, slots] = _exact_quantised(state[name][s, which])
            out[name] = (values, powers)
        return [out["k"][0], out["v"][0], out["k"][1], out["v"][1]]
    if kind == "read":
        out = [state["k_out"].double(), state["v_out"].double()]
        for s, n in enumerate(lengths):
            start = 0 if state["starts"] is None else int(state["starts"][s])
            upto = max(start, min(n, start + out[0].shape[1]))
            for values, name in zip(out, ("k", "v")):
                values[s, :upto - start] = token_values(name, s, torch.arange(start, upto, device="cuda"))
        return out
    q, tree = state["q"].double(), state["tree"].cpu()
    b, t, h, d = q.shape
    kv = state["k"].shape[2]
    group, out = h // kv, torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
    for s, n in enumerate(lengths):
        where = torch.arange(n, device="cuda")
        sees = torch.tensor([[(int(word) >> j) & 1 for j in range(t)] for word in tree[s]], dtype=torch.bool, device="cuda")
        allowed = torch.cat([sees.any(1, keepdim=True).expand(t, n), sees], 1)
        keys, values = (torch.cat([token_values(name, s, where), state[name][s].double()]) for name in ("k", "v"))
        for g in range(kv):
            scores = torch.einsum("tgd,sd->tgs", q[s, :, g * group:(g + 1) * group], keys[:, g]) * d ** -0.5
            scores = torch.where(allowed[:, None, :], scores, -math.inf)
            out[s, :, g * group:(g + 1) * group] = torch.einsum("tgs,sd->tgd", torch.softmax(scores, 2).nan_to_num(0.0), values[:, g])
    return out


def work(case):
    kind = case["kind"]
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["type"]]
    if kind == "verify":
        # the rows of the last accepted token; of the tokens before it a few values each
        b, t, vocab = case["b"], case["t"], case["vocab"]
        rows = 2 if case["draft"] and t > 1 else 1
        return {"bytes": b * vocab * size * rows + b * t * 28 + 12 * b, "flops": b * vocab * (2 + 3 * (rows - 1))}
    kv, d = case["kv"], case["d"]
    if kind == "write":
        rows = 2 * case["b"] * kv * (case["t"] if not case["take"] else (case["t"] + 1) // 2)
        return {"bytes": rows * (3 * d + 1), "flops": rows * 3 * d}
    tokens = sum(_lengths(case))
    if kind == "read":
        rows = 2 * kv * (tokens // 3 if case["part"] else tokens)
        return {"bytes": rows * (3 * d + 1) + 4 * tokens // case["page"], "flops": rows * d}
    b, t, h = case["b"], case["t"], case["heads"]
    return {"bytes": 2 * (d + 1) * kv * tokens + 4 * d * kv * b * t + 4 * d * h * b * t + 4 * tokens // case["page"] + 8 * b * t,
            "flops": 4 * d * h * t * (tokens + b * (t + 1) // 2)}
