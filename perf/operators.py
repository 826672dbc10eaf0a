"""The operators that stand between the weight products of a decoder block, as cases that can be timed.

Root-mean-square norm with the residual's addition (16-bit output, or E4M3 with a scale for each 128 neighbours of a row), the
product of two E4M3 matrices with such scales, and attention of a tree of drafted tokens over a paged cache.  With ``own`` the
calls are those of ``fp6_marlin_b200``; without it the same formulas in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
SMALLEST = 1e-30                  # a group of zeros gets this as its largest magnitude
GROUP = 128

MOST_MUL_FLOPS = 2 * 4096 * 8192 * 28672
MOST_NORM_VALUES = 16384 * 8192
MOST_KV_TOKENS = 64 * 8 * 6144    # tokens of the cache x heads of keys and values
MOST_SCORES = 2 * 64 * 64 * 32768 # query heads x drafted tokens x keys


def listed():
    return [
        # one token's residual stream between two layers of a 7B block: launch and latency only
        {"name": "norm m1 n4096", "kind": "norm", "m": 1, "n": 4096, "type": "f16", "residual": True, "fp8": False},
        # prefill of a long batch: the norm as a stream through memory
        {"name": "norm fp8 m16384 n8192", "kind": "norm", "m": 16384, "n": 8192, "type": "f16", "residual": True, "fp8": True},
        # the attention's output for a tree of drafted tokens of a 70B model, on its way into an 8-bit output projection
        {"name": "quantise m37 n8192", "kind": "quantise", "m": 37, "n": 8192, "type": "bf16"},
        # the activations of a feed-forward layer, rounded to 8 bits in front of the 7B down projection, a batch of odd length
        {"name": "quantise m4099 n11008", "kind": "quantise", "m": 4099, "n": 11008, "type": "f16"},
        # one token through a square projection: latency
        {"name": "fp8 4096x4096 m1", "kind": "mul", "m": 1, "k": 4096, "n": 4096, "type": "f16"},
        # the largest decode layer, the 70B gate / up projection, half a gigabyte of weights
        {"name": "fp8 8192x57344 m16", "kind": "mul", "m": 16, "k": 8192, "n": 57344, "type": "bf16"},
        # a tree for each of a few sequences through the 7B down projection, no multiple of a tile
        {"name": "fp8 11008x4096 m131", "kind": "mul", "m": 131, "k": 11008, "n": 4096, "type": "f16"},
        # compute-bound prefill through half of the 70B gate / up projection
        {"name": "fp8 8192x28672 m4096", "kind": "mul", "m": 4096, "k": 8192, "n": 28672, "type": "f16"},
        # the next token of one short sequence, a head of keys for each head of queries: latency
        {"name": "decode b1 t1 32/32 l300", "kind": "tree", "b": 1, "t": 1, "heads": 32, "kv": 32, "d": 128, "cache": 300, "page": 16, "type": "f16", "even": False},
        # small trees over the ragged caches of a few sequences
        {"name": "tree b8 t5 32/32 l4096", "kind": "tree", "b": 8, "t": 5, "heads": 32, "kv": 32, "d": 128, "cache": 4096, "page": 64, "type": "f16", "even": False},
        # a large tree over two long caches, eight heads of queries to each head of keys: 512 rows share a key
        {"name": "tree b2 t64 64/8 l32768", "kind": "tree", "b": 2, "t": 64, "heads": 64, "kv": 8, "d": 128, "cache": 32768, "page": 16, "type": "bf16", "even": True},
        # a serving batch, a few drafted tokens each
        {"name": "tree b64 t7 64/8 l6144", "kind": "tree", "b": 64, "t": 7, "heads": 64, "kv": 8, "d": 128, "cache": 6144, "page": 48, "type": "bf16", "even": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _multiple(rng, lo, hi, of):
    while True:
        n = max(1, round(_log_int(rng, lo, hi) / of)) * of
        if n != 3072:
            return n


def draw(rng):
    pick, kind_of = rng.random(), rng.choice(["f16", "bf16"])
    if pick < 0.25:
        while True:
            m, n = _log_int(rng, 1, 16384), _multiple(rng, 512, 16384, 8)
            if m * n <= MOST_NORM_VALUES:
                break
        if rng.random() < 0.3:
            return {"kind": "quantise", "m": m, "n": n, "type": kind_of}
        return {"kind": "norm", "m": m, "n": n, "type": kind_of, "residual": rng.random() < 0.7, "fp8": rng.random() < 0.6}
    if pick < 0.62:
        while True:
            m, k, n = _log_int(rng, 1, 4096), _multiple(rng, 512, 16384, 16), _multiple(rng, 512, 57344, 8)
            if 2 * m * k * n <= MOST_MUL_FLOPS and k * n <= 8192 * 57344:
                return {"kind": "mul", "m": m, "k": k, "n": n, "type": kind_of}
    while True:
        b, t, kv, group = _log_int(rng, 1, 64), _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 5, 8])
        case = {"kind": "tree", "b": b, "t": t, "heads": kv * group, "kv": kv, "d": rng.choice([64, 128, 128]), "cache": _log_int(rng, 16, 32768),
                "page": rng.choice([1, 16, 16, 24, 32, 64, 128, 256]), "type": kind_of, "even": rng.random() < 0.3}
        if b * kv * case["cache"] <= MOST_KV_TOKENS and b * t * kv * group * (case["cache"] + t) <= MOST_SCORES and kv * group <= 64:
            return case


def _lengths(case):
    """Committed tokens of each sequence: all alike, or ragged from an empty cache to the longest."""
    b, longest = case["b"], case["cache"]
    if case["even"] or b == 1:
        return [longest] * b
    return [longest * i // (b - 1) for i in range(b)]


def _type(case):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[case["type"]]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _stream_of_activations(gen, m, n, dtype):
    # a residual stream: unit variance with a few channels that are much larger
    loud = torch.ones(n, device="cuda")
    loud[torch.randint(n, (max(1, n // 512),), generator=gen, device="cuda")] = 20.0
    return (_randn(gen, m, n) * loud).to(dtype)


def _quantised_rows(x):
    m, n = x.shape
    groups = -(-n // GROUP)
    s = torch.nn.functional.pad(x, (0, groups * GROUP - n)).view(m, groups, GROUP).abs().amax(2).clamp(min=SMALLEST) / E4M3_MAX
    q = (x / s.repeat_interleave(GROUP, 1)[:, :n]).to(torch.float8_e4m3fn)
    return q, s


def _quantised_weight(gen, n, k):
    nb, kb = -(-n // GROUP), -(-k // GROUP)
    w = torch.empty((n, k), dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty((nb, kb), device="cuda")
    part = 64 * GROUP             # rows at a time: 32-bit copies of a large layer stay small
    for at in range(0, n, part):
        rows = min(part, n - at)
        x = torch.randn((rows, k), generator=gen, device="cuda") * 0.02
        blocks = torch.nn.functional.pad(x, (0, kb * GROUP - k, 0, -rows % GROUP)).view(-1, GROUP, kb, GROUP)
        sb = blocks.abs().amax((1, 3)).clamp(min=SMALLEST) / E4M3_MAX
        w[at:at + rows] = (blocks / sb[:, None, :, None]).view(-1, kb * GROUP)[:rows, :k].to(torch.float8_e4m3fn)
        s[at // GROUP:at // GROUP + sb.shape[0]] = sb
    return w, s


def _trees(gen, b, t):
    """Random trees: the first token hangs on the last committed one, every other on an earlier drafted token or beside the first."""
    parent = (torch.rand((b, t), generator=gen) * torch.arange(t)).long() - 1
    parent = torch.where(torch.rand((b, t), generator=gen) < 0.5, torch.arange(t).expand(b, t) - 1, parent)
    see = torch.zeros((b, t, t), dtype=torch.bool)
    for i in range(t):
        p = parent[:, i]
        see[:, i] = torch.where((p >= 0)[:, None], see[torch.arange(b), p.clamp(min=0)], False)
        see[:, i, i] = True
    if b > 2 and t > 2:
        see[1, t - 1] = False     # a sequence with one token fewer: its last place is padding
        see[1, :, t - 1] = False
    return (see.long() << torch.arange(t)).sum(2).cuda()


def prepare(case, seed):
    gen, kind, dtype = torch.Generator(device="cuda").manual_seed(seed), case["kind"], _type(case)
    if kind in ("norm", "quantise"):
        m, n = case["m"], case["n"]
        state = {"kind": kind, "x": _stream_of_activations(gen, m, n, dtype), "eps": 1e-6}
        fp8 = kind == "quantise" or case["fp8"]
        state["y"] = torch.empty((m, n), dtype=torch.float8_e4m3fn if fp8 else dtype, device="cuda")
        state["scales"] = torch.empty((m, -(-n // GROUP)), device="cuda") if fp8 else None
        if kind == "norm":
            state["weight"] = (1 + 0.2 * _randn(gen, n)).to(dtype)
            state["residual"] = _stream_of_activations(gen, m, n, dtype) if case["residual"] else None
            state["sum"] = torch.empty((m, n), dtype=dtype, device="cuda") if case["residual"] else None
        return state
    if kind == "mul":
        m, k, n = case["m"], case["k"], case["n"]
        a, sa = _quantised_rows(_stream_of_activations(gen, m, k, torch.float32))
        w, sb = _quantised_weight(gen, n, k)
        return {"kind": kind, "a": a, "sa": sa, "b": w, "sb": sb, "c": torch.empty((m, n), dtype=dtype, device="cuda")}
    b, t, h, kv, d, page = (case[x] for x in ("b", "t", "heads", "kv", "d", "page"))
    host = torch.Generator().manual_seed(seed)
    lengths = torch.tensor(_lengths(case))[torch.randperm(b, generator=host)]
    per = -(-max(case["cache"], 1) // page)
    pages = b * per
    # the projection's output: queries, keys and values of a token next to one another
    qkv = _randn(gen, b, t, (h + 2 * kv) * d)
    qkv[..., :h * d] *= 2
    qkv = qkv.to(dtype)
    return {"kind": kind, "q": qkv[..., :h * d].unflatten(2, (h, d)), "k": qkv[..., h * d:(h + kv) * d].unflatten(2, (kv, d)),
            "v": qkv[..., (h + kv) * d:].unflatten(2, (kv, d)),
            "k_cache": torch.randn((pages, page, kv, d), generator=gen, device="cuda", dtype=dtype),
            "v_cache": torch.randn((pages, page, kv, d), generator=gen, device="cuda", dtype=dtype),
            "pages": torch.randperm(pages, generator=host).view(b, per).int().cuda(), "lengths": lengths.int().cuda(), "tree": _trees(host, b, t),
            "out": torch.empty((b, t, h, d), dtype=dtype, device="cuda")}


def _run_own(state):
    import fp6_marlin_b200 as fm
    kind = state["kind"]
    if kind == "norm":
        fm.rms_norm(state["x"], state["weight"], state["y"], state["eps"], scales=state["scales"], residual=state["residual"], residual_out=state["sum"])
        return [state["y"], state["scales"], state["sum"]]
    if kind == "quantise":
        fm.quantize_fp8(state["x"], state["y"], state["scales"])
        return [state["y"], state["scales"]]
    if kind == "mul":
        fm.mul_fp8(state["a"], state["b"], state["c"], state["sa"], state["sb"])
        return state["c"]
    fm.tree_attention(state["q"], state["k"], state["v"], state["k_cache"], state["v_cache"], state["pages"], state["lengths"], state["tree"], state["out"])
    return state["out"]


def _attend(q, k, v, k_cache, v_cache, pages, lengths, tree):
    b, t, h, d = q.shape
    kv, longest = k.shape[2], pages.shape[1] * k_cache.shape[1]
    cached = torch.arange(longest, device=q.device) < lengths[:, None]                                                  # b, longest
    sees = (tree[:, :, None] >> torch.arange(t, device=q.device)) & 1 != 0                                              # b, t, t
    real = tree != 0
    visible = torch.cat([(cached[:, None, :] & real[:, :, None]), sees], 2)                                              # b, t, longest + t
    keys = torch.cat([k_cache[pages.long()].view(b, longest, kv, d), k], 1).float()
    values = torch.cat([v_cache[pages.long()].view(b, longest, kv, d).masked_fill(~cached[:, :, None, None], 0), v], 1).float()
    rows = q.float().view(b, t, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, t * (h // kv), d)
    scores = (rows @ keys.permute(0, 2, 3, 1)).view(b, kv, t, h // kv, -1) / math.sqrt(d)
    scores = scores.masked_fill_(~visible[:, None, :, None, :], -math.inf)
    top = scores.amax(4, keepdim=True).clamp(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(4, keepdim=True)
    out = (p.view(b, kv, t * (h // kv), -1) @ values.transpose(1, 2)).view(b, kv, t, h // kv, d) / total.clamp(min=1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, h, d)


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind in ("norm", "quantise"):
        y, total = state["x"].float(), None
        if kind == "norm":
            if state["residual"] is not None:
                y = y + state["residual"].float()
                total = y.to(state["x"].dtype)
            y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + state["eps"]) * state["weight"].float()
        if state["scales"] is None:
            return [y.to(state["x"].dtype), None, total]
        q, s = _quantised_rows(y)
        return [q, s, total] if kind == "norm" else [q, s]
    if kind == "mul":
        a = state["a"].float() * state["sa"].repeat_interleave(GROUP, 1)[:, :state["a"].shape[1]]
        n, k = state["b"].shape
        w = state["b"].float() * state["sb"].repeat_interleave(GROUP, 1)[:, :k].repeat_interleave(GROUP, 0)[:n]
        return (a @ w.T).to(state["c"].dtype)
    return _attend(*(state[x] for x in ("q", "k", "v", "k_cache", "v_cache", "pages", "lengths", "tree"))).to(state["out"].dtype)


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    if kind in ("norm", "quantise"):
        y, total = state["x"].double(), None
        if kind == "norm":
            if state["residual"] is not None:
                y = total = y + state["residual"].double()
            y = y / ((y * y).sum(1) / y.shape[1] + state["eps"]).sqrt()[:, None] * state["weight"].double()
        if state["scales"] is None:
            return [y, None, total]
        m, n = y.shape
        at = torch.arange(n, device=y.device) // GROUP
        s = torch.zeros((m, int(at[-1]) + 1), dtype=torch.float64, device=y.device).scatter_reduce_(1, at.expand(m, n), y.abs(), "amax")
        s = torch.maximum(s, torch.tensor(SMALLEST, dtype=torch.float64, device=y.device)) / E4M3_MAX
        q = y / s[:, at]          # before it is rounded to eight bits
        return [q, s, total] if kind == "norm" else [q, s]
    if kind == "mul":
        a, w, sa, sb = state["a"].double(), state["b"], state["sa"].double(), state["sb"].double()
        c = torch.zeros((a.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
        column = torch.arange(w.shape[0], device="cuda") // GROUP
        for g in range(sa.shape[1]):
            block = slice(g * GROUP, (g + 1) * GROUP)
            c += (a[:, block] * sa[:, g:g + 1]) @ (w[:, block].double() * sb[column, g][:, None]).T
        return c
    q, k, v, tree, page = state["q"].double(), state["k"].double(), state["v"].double(), state["tree"].cpu(), state["k_cache"].shape[1]
    b, t, h, d = q.shape
    group, out = h // k.shape[2], torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
    for i, length in enumerate(state["lengths"].tolist()):
        where = torch.arange(length, device="cuda")
        page_of, slot = state["pages"][i].long()[where // page], where % page
        sees = torch.tensor([[(int(word) >> j) & 1 for j in range(t)] for word in tree[i]], dtype=torch.bool, device="cuda")
        allowed = torch.cat([sees.any(1, keepdim=True).expand(t, length), sees], 1)
        for g in range(k.shape[2]):
            keys = torch.cat([state["k_cache"][page_of, slot, g].double(), k[i, :, g]])
            values = torch.cat([state["v_cache"][page_of, slot, g].double(), v[i, :, g]])
            scores = torch.einsum("tgd,sd->tgs", q[i, :, g * group:(g + 1) * group], keys) * d ** -0.5
            scores = torch.where(allowed[:, None, :], scores, -math.inf)
            p = torch.softmax(scores, 2).nan_to_num(0.0)
            out[i, :, g * group:(g + 1) * group] = torch.einsum("tgs,sd->tgd", p, values)
    return out


def work(case):
    kind = case["kind"]
    if kind in ("norm", "quantise"):
        m, n = case["m"], case["n"]
        fp8, residual = kind == "quantise" or case["fp8"], kind == "norm" and case["residual"]
        nbytes = 2 * m * n + (2 * n if kind == "norm" else 0) + (4 * m * n if residual else 0) + (m * n + 4 * m * -(-n // GROUP) if fp8 else 2 * m * n)
        return {"bytes": nbytes, "flops": m * n * (6 if kind == "norm" else 2)}
    if kind == "mul":
        m, k, n = case["m"], case["k"], case["n"]
        kb, nb = -(-k // GROUP), -(-n // GROUP)
        return {"bytes": n * k + m * k + 4 * kb * (m + nb) + 2 * m * n, "flops": 2 * m * n * k}
    b, t, h, kv, d = (case[x] for x in ("b", "t", "heads", "kv", "d"))
    tokens = sum(_lengths(case))
    return {"bytes": 4 * d * kv * (tokens + b * t) + 4 * d * h * b * t + 4 * tokens // case["page"] + 8 * b * t,
            "flops": 4 * d * h * t * (tokens + b * (t + 1) // 2)}
