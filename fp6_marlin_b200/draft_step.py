"""One decoder block over trees of drafted tokens: the operators of this package as they follow one another.

    python -m fp6_marlin_b200.draft_step [--sequences 8] [--tokens 16] [--cached 2048] [--fp8-cache]

A block of a 7B model with random weights.  The queries / keys / values and gate / up projections are kept in 8 bits, the output and
down projections in INT4 / FP6.  A step takes the drafted tokens of every sequence through the block:

    rms_norm -> E4M3 -> mul_fp8 (qkv) -> rotary positions -> tree_attention over the paged cache -> mul (output projection)
    -> rms_norm with the residual's addition -> E4M3 -> mul_fp8 (gate, up) -> silu * up -> mul_fused (down projection + residual)

What the drafted tokens are not needed for any more once some are accepted - their keys and values - then goes into the cache
(:meth:`DraftBlock.accept`).  With a cache in 8 bits (``fp8_cache``, and ``vocab`` for a projection onto a vocabulary) the step is closed on the device:

    ... -> tree_attention_fp8 -> ... -> rms_norm -> mul_fp8 (vocabulary) -> softmax -> verify_drafts -> write_cache_fp8 of the accepted tokens

(:meth:`DraftBlock.choose`, :meth:`DraftBlock.commit`), with no synchronisation, so that all of it can be captured in a CUDA graph.  The program prints the time of a step and
the relative error of its result against the same step in elementary torch operations.
"""
from __future__ import annotations

import argparse

import torch

from .api import mul, mul_fused
from .block_ops import GROUP, make_fp8_weight, mul_fp8, rms_norm, tree_attention, tree_masks
from .decode_ops import make_cache_fp8, tree_attention_fp8, verify_drafts, write_cache_fp8
from .quant import make_w46_weight


class DraftBlock:
    """Weights, cache and work buffers of one decoder block for up to ``sequences * tokens`` rows at a time."""

    def __init__(self, hidden=4096, inter=11008, heads=32, kv_heads=32, sequences=8, tokens=16, pages=1024, page_size=16, quant_cols=256, seed=0, device="cuda", fp8_cache=False, vocab=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        randn = lambda *shape: torch.randn(shape, generator=gen, device=device)          # noqa: E731
        self.heads, self.kv_heads, self.dim = heads, kv_heads, hidden // heads
        self.sequences, self.tokens, self.quant_cols, self.vocab = sequences, tokens, quant_cols, vocab
        self.norm1, self.norm2 = ((1 + 0.1 * randn(hidden)).half() for _ in range(2))
        self.qkv = make_fp8_weight(randn((heads + 2 * kv_heads) * self.dim, hidden) * 0.02)
        self.gate_up = make_fp8_weight(randn(2 * inter, hidden) * 0.02)
        self.out = make_w46_weight((randn(hidden, hidden) * 0.02).half(), quant_cols, GROUP, quant_device=device)
        self.down = make_w46_weight((randn(inter, hidden) * 0.02).half(), quant_cols, GROUP, quant_device=device)
        self.k_cache, self.v_cache = (randn(pages, page_size, kv_heads, self.dim).half() for _ in range(2))
        self.fp8 = None
        if fp8_cache:
            # the same values in 8 bits: every page is written as the first tokens of a sequence of its own
            self.fp8 = make_cache_fp8(pages, page_size, kv_heads, self.dim, device)
            write_cache_fp8(self.k_cache, self.v_cache, *self.fp8, torch.arange(pages, dtype=torch.int32, device=device)[:, None], torch.zeros(pages, dtype=torch.int32, device=device))
            self.k_cache = self.v_cache = None
        rows, half = sequences * tokens, dict(dtype=torch.float16, device=device)
        if vocab:
            self.norm3, self.head = (1 + 0.1 * randn(hidden)).half(), make_fp8_weight(randn(vocab, hidden) * 0.05)
            self.logits = torch.empty((rows, vocab), **half)
            self.accepted, self.counts = (torch.empty(shape, dtype=torch.int32, device=device) for shape in ((sequences, tokens), (sequences,)))
            self.next_tokens = torch.empty(sequences, dtype=torch.int64, device=device)
        self.rows8, self.scales = torch.empty((rows, hidden), dtype=torch.float8_e4m3fn, device=device), torch.empty((rows, -(-hidden // GROUP)), device=device)
        self.qkv_out = torch.empty((rows, self.qkv[0].shape[0]), **half)
        self.gate_up_out, self.act = torch.empty((rows, 2 * inter), **half), torch.empty((rows, inter), **half)
        self.attended, self.projected, self.stream, self.result = (torch.empty((rows, hidden), **half) for _ in range(4))
        self.workspace = torch.zeros(max(hidden, 2 * inter) // 128 * 16, dtype=torch.int32, device=device)
        self.angles = 10000.0 ** (-torch.arange(0, self.dim, 2, device=device) / self.dim)

    def _rotate(self, x, positions):
        """Rotary positions of x (sequences, tokens, heads, dim), in fp32."""
        angle = positions[..., None, None] * self.angles
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1).half()

    def step(self, x, page_table, lengths, tree):
        """x (sequences * tokens, hidden) fp16 through the block; tree: the masks of :func:`tree_masks`.  Returns (result, keys, values)."""
        b, t, h, g, d = self.sequences, self.tokens, self.heads, self.kv_heads, self.dim
        rms_norm(x, self.norm1, self.rows8, scales=self.scales)
        mul_fp8(self.rows8, self.qkv[0], self.qkv_out, self.scales, self.qkv[1])
        q, k, v = self.qkv_out.view(b, t, h + 2 * g, d).split([h, g, g], 2)
        bits = torch.arange(t, device=x.device)
        depth = ((tree[..., None] >> bits) & 1).sum(-1) - 1                       # ancestors of a drafted token
        positions = (lengths[:, None] + depth).float()
        q, k = self._rotate(q, positions), self._rotate(k, positions)
        attended = self.attended.view(b, t, h, d)
        if self.fp8 is None:
            tree_attention(q, k, v, self.k_cache, self.v_cache, page_table, lengths, tree, attended)
        else:
            tree_attention_fp8(q, k, v, *self.fp8, page_table, lengths, tree, attended)
        mul(self.attended, self.out.B, self.projected, self.out.s, self.workspace, self.quant_cols, group_size=GROUP, layout="b200")
        rms_norm(self.projected, self.norm2, self.rows8, scales=self.scales, residual=x, residual_out=self.stream)
        mul_fp8(self.rows8, self.gate_up[0], self.gate_up_out, self.scales, self.gate_up[1])
        gate, up = self.gate_up_out.float().chunk(2, 1)
        self.act.copy_(torch.nn.functional.silu(gate) * up)
        mul_fused(self.act, self.down.B, self.result, self.down.s, self.workspace, self.quant_cols, epilogue="residual", residual=self.stream, group_size=GROUP)
        return self.result, k, v

    def choose(self, result, drafted, tree, uniforms, draft=None):
        """From the rows of a step to the accepted drafted tokens: ``(accepted, counts, next_tokens)`` as :func:`verify_drafts` gives them.  The target's probabilities are the softmax
        of a projection onto the vocabulary in 8 bits; drafted (sequences, tokens): the ids; uniforms: random numbers; draft: the probabilities that the ids were drawn from."""
        if not self.vocab:
            raise ValueError("choose: a block with vocab= is needed")
        rms_norm(result, self.norm3, self.rows8, scales=self.scales)
        mul_fp8(self.rows8, self.head[0], self.logits, self.scales, self.head[1])
        target = torch.softmax(self.logits.float(), 1).view(self.sequences, self.tokens, -1)
        verify_drafts(target, drafted, tree, uniforms, self.accepted, self.counts, self.next_tokens, draft=draft)
        return self.accepted, self.counts, self.next_tokens

    def commit(self, keys, values, accepted, counts, page_table, lengths):
        """Writes the keys and values of the accepted drafted tokens into the 8-bit cache, behind the committed ones, and counts them into ``lengths``, all on the device.  The page table must have
        places for them: what has none is not written and reported by ``device_status`` (4), and ``lengths`` go up to the first such token only."""
        if self.fp8 is None:
            raise ValueError("commit: a 16-bit cache is written by accept")
        write_cache_fp8(keys, values, *self.fp8, page_table, lengths, tokens=accepted, counts=counts)
        places, (pages, page_size) = page_table.shape[1], self.fp8[0].shape[:2]
        if not places:
            return
        entry = torch.arange(accepted.shape[1], device=keys.device)
        place = (lengths.long()[:, None] + entry) // page_size
        page = page_table.gather(1, place.clamp(0, places - 1))
        written = (entry < counts[:, None]) & (accepted >= 0) & (accepted < keys.shape[1]) & (place < places) & (page >= 0) & (page < pages)
        lengths += written.int().cumprod(1).sum(1)

    def cached_values(self):
        """The cache's keys and values in fp32."""
        if self.fp8 is None:
            return self.k_cache.float(), self.v_cache.float()
        return tuple(c.float() * torch.exp2(e.float() - 127)[..., None] for c, e in zip(self.fp8[:2], self.fp8[2:]))

    def accept(self, keys, values, accepted, page_table, lengths):
        """Writes the keys and values of accepted drafted tokens (``accepted``: a list of token numbers per sequence) behind the
        committed ones and returns the new lengths.  Raises ``ValueError``, and writes nothing, where there is no such token or no place for it
        (this check synchronises; on the GPU an index out of range would end the process's use of it)."""
        if self.k_cache is None:
            raise ValueError("accept: a cache in 8 bits is written by commit")
        page_size = self.k_cache.shape[1]
        if not len(accepted) == keys.shape[0] == lengths.shape[0] == page_table.shape[0] or any(not 0 <= t < keys.shape[1] for tokens in accepted for t in tokens):
            raise ValueError("accept: a list of numbers of drafted tokens for each sequence is needed")
        index = lambda values: torch.tensor(values, dtype=torch.long, device=keys.device)          # noqa: E731  (also of none)
        sequence = index([i for i, tokens in enumerate(accepted) for _ in tokens])
        token = index([t for tokens in accepted for t in tokens])
        rank = index([j for tokens in accepted for j in range(len(tokens))])
        at = lengths.long()[sequence] + rank
        place, slot = (at // page_size).clamp(0, max(page_table.shape[1] - 1, 0)), at % page_size
        page = page_table.long()[sequence, place] if page_table.shape[1] else torch.full_like(at, -1)
        if bool(((place != at // page_size) | (page < 0) | (page >= self.k_cache.shape[0])).any()):
            raise ValueError("accept: the page table has no place for an accepted token")
        self.k_cache[page, slot], self.v_cache[page, slot] = keys[sequence, token], values[sequence, token]
        return lengths + torch.tensor([len(tokens) for tokens in accepted], dtype=torch.int32, device=keys.device)


def plain_step(block: DraftBlock, x, page_table, lengths, tree):
    """The same step in elementary torch operations in fp32, with the same roundings of rows to E4M3."""
    def rows8(y):
        s = torch.nn.functional.pad(y, (0, -y.shape[1] % GROUP)).view(y.shape[0], -1, GROUP).abs().amax(2).clamp(min=1e-30) / 448
        s = s.repeat_interleave(GROUP, 1)[:, : y.shape[1]]
        return (y / s).to(torch.float8_e4m3fn).float() * s

    def norm(y, w):
        return y * torch.rsqrt(y.square().mean(1, keepdim=True) + 1e-6) * w.float()

    def weight8(pair):
        return pair[0].float() * pair[1].repeat_interleave(GROUP, 0)[: pair[0].shape[0]].repeat_interleave(GROUP, 1)[:, : pair[0].shape[1]]

    b, t, h, g, d = block.sequences, block.tokens, block.heads, block.kv_heads, block.dim
    q, k, v = (rows8(norm(x.float(), block.norm1)) @ weight8(block.qkv).T).view(b, t, h + 2 * g, d).split([h, g, g], 2)
    sees = (tree[..., None] >> torch.arange(t, device=x.device)) & 1 != 0
    positions = (lengths[:, None] + sees.sum(-1) - 1).float()
    q, k = block._rotate(q, positions).float(), block._rotate(k, positions).float()
    attended = torch.empty((b, t, h, d), device=x.device)
    k_cache, v_cache = block.cached_values()
    for i, n in enumerate(lengths.tolist()):
        keys, values = (torch.cat([c[page_table[i].long()].flatten(0, 1)[:n], new[i]]).repeat_interleave(h // g, 1) for c, new in ((k_cache, k), (v_cache, v)))
        scores = torch.einsum("thd,nhd->thn", q[i], keys) * d ** -0.5
        scores[..., n:].masked_fill_(~sees[i][:, None], -torch.inf)
        attended[i] = torch.einsum("thn,nhd->thd", scores.softmax(-1), values)
    stream = x.float() + attended.view(b * t, h * d) @ block.out.w_deq.to(x.device).float()
    gate, up = (rows8(norm(stream, block.norm2)) @ weight8(block.gate_up).T).chunk(2, 1)
    return stream + (torch.nn.functional.silu(gate) * up) @ block.down.w_deq.to(x.device).float()


def make_inputs(block: DraftBlock, cached: int, seed=0):
    """Rows, page table, ragged lengths and random trees for a step."""
    cache = block.k_cache if block.fp8 is None else block.fp8[0]
    gen, device = torch.Generator().manual_seed(seed), cache.device
    b, t, page_size = block.sequences, block.tokens, cache.shape[1]
    per = -(-(cached + t) // page_size)
    page_table = torch.randperm(cache.shape[0], generator=gen)[: b * per].view(b, per).int().to(device)
    lengths = torch.tensor([cached * (i + 1) // b for i in range(b)], dtype=torch.int32, device=device)
    parents = (torch.rand((b, t), generator=gen) * torch.arange(t)).long() - 1
    return torch.randn((b * t, block.norm1.numel()), generator=gen).half().to(device), page_table, lengths, tree_masks(parents).to(device)


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--sequences", type=int, default=8)
    parser.add_argument("--tokens", type=int, default=16)
    parser.add_argument("--cached", type=int, default=2048)
    parser.add_argument("--fp8-cache", action="store_true", help="a cache in 8 bits, and the choice among the drafted tokens")
    options = parser.parse_args()
    per = -(-(options.cached + options.tokens) // 16)
    block = DraftBlock(sequences=options.sequences, tokens=options.tokens, pages=options.sequences * per, fp8_cache=options.fp8_cache, vocab=32000 if options.fp8_cache else 0)
    x, page_table, lengths, tree = make_inputs(block, options.cached)
    result, keys, values = block.step(x, page_table, lengths, tree)
    expect = plain_step(block, x, page_table, lengths, tree)
    print(f"{options.sequences} sequences x {options.tokens} drafted tokens over up to {options.cached} cached ones: relative error "
          f"{float((result.float() - expect).norm() / expect.norm()):.2e}")
    if options.fp8_cache:
        gen = torch.Generator(device="cuda").manual_seed(1)
        drafted = torch.randint(32000, tree.shape, generator=gen, device="cuda")
        uniforms = torch.rand(tree.shape, generator=gen, device="cuda")

    def whole_step():
        result, keys, values = block.step(x, page_table, lengths, tree)
        return (*block.choose(result, drafted, tree, uniforms), keys, values) if options.fp8_cache else (keys, values)

    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(3):
        whole_step()
    start.record()
    for _ in range(20):
        *chosen, keys, values = whole_step()
    end.record()
    torch.cuda.synchronize()
    print(f"a step: {start.elapsed_time(end) * 50:.0f} us")
    if options.fp8_cache:
        accepted, counts, next_tokens = chosen
        block.commit(keys, values, accepted, counts, page_table, lengths)
        print("accepted tokens:", counts.tolist(), "next:", next_tokens.tolist(), "lengths:", lengths.tolist())
    else:
        lengths = block.accept(keys, values, [[0]] * options.sequences, page_table, lengths)
        print("lengths with one accepted token each:", lengths.tolist())


if __name__ == "__main__":
    main()
