"""What decoding with drafted tokens needs around attention: a paged cache in 8 bits, attention over it, the choice among drafted tokens.

``write_cache_fp8`` puts the keys and values of new or accepted tokens into a cache of E4M3 values with a power of two for each token and head,
``read_cache_fp8`` brings them back in 16 bits, ``tree_attention_fp8`` is ``tree_attention`` over such a cache, which has half the bytes,
and ``verify_drafts`` decides from the target's probabilities which drafted tokens are accepted and which token follows.  Accepted tokens' numbers and
their counts stay on the device and are what ``write_cache_fp8`` takes, so that a step of decoding needs no synchronisation and can be captured in a CUDA
graph.  As in ``block_ops`` outputs are tensors of the caller that are overwritten, and all calls run asynchronously on the current stream of their
device.  The reference has no counterpart of these; its layer lists (bench.py:53-86) name the products on either side.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .api import _call, _device_buffers, _ptr, _status, _stream_handle
from .block_ops import _TYPES, _buffers_lock, _operator_buffers, _raise, _sms, _strides, _tree_args
from ._lib import lib

_PROBABILITIES = {**_TYPES, torch.float32: _lib.TYPE_F32}


def make_cache_fp8(pages, page_size, kv_heads, head_dim, device="cuda"):
    """An empty cache: ``(k_cache, v_cache, k_scales, v_scales)``, float8_e4m3fn (pages, page_size, kv_heads, head_dim) and uint8
    (pages, page_size, kv_heads).  A byte holds the exponent of its head's power of two, plus 127; those of a page lie head by head."""
    caches = [torch.zeros((pages, page_size, kv_heads, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    return (*caches, *(torch.full((pages, kv_heads, page_size), 127, dtype=torch.uint8, device=device).transpose(1, 2) for _ in range(2)))


def _scales(what, k_scales, v_scales, shape, device, written=False):
    strides = []
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if t.dtype != torch.uint8 or tuple(t.shape) != shape:
            raise RuntimeError(f"{what}: {name} must be uint8 of shape {shape}")
        if t.device != device:
            raise RuntimeError(f"{what}: {name} must be on the same CUDA device as the other tensors")
        s = [1 if size == 1 else step for size, step in zip(shape, t.stride())]
        if written and any(size > 1 and step == 0 for size, step in zip(shape, s)):
            raise RuntimeError(f"{what}: places of {name} share memory")
        strides.append((ctypes.c_longlong * 3)(*s))
    return _lib.CacheScales(_ptr(k_scales), _ptr(v_scales), *strides)


def _ints(what, name, t, shape, device):
    """An optional int32 tensor whose rows are contiguous; its address."""
    if t is None:
        return 0
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise RuntimeError(f"{what}: {name} must be int32 of shape {shape}")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} must be on the same CUDA device as the other tensors")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise RuntimeError(f"{what}: the rows of {name} must be contiguous")
    return _ptr(t)


def _move(what, function, k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, written, entries, **lists):
    if not k.is_cuda:
        raise RuntimeError(f"fp6_marlin_b200.{what} needs CUDA tensors: there is no CPU implementation")
    if k.dtype not in _TYPES or k.dim() != 4 or k_cache.dim() != 4 or page_table.dim() != 2:
        raise RuntimeError(f"{what}: k and v must be (B, tokens, heads, head size) of float16 or bfloat16, the cache (pages, page size, heads, head size) and the page table (B, P)")
    b, t, g, d = k.shape
    if d not in (64, 128):
        raise RuntimeError(f"{what}: heads of 64 or 128 values")
    pages, page_size = k_cache.shape[:2]
    device, place, into = k.device, (pages, page_size, g, d), written == "cache"
    scales = _scales(what, k_scales, v_scales, place[:3], device, into)
    wide = [_strides(what, name, x, k.dtype, (b, t, g, d), device, not into) for name, x in (("k", k), ("v", v))]
    cache = [_strides(what, name, x, torch.float8_e4m3fn, place, device, into) for name, x in (("k_cache", k_cache), ("v_cache", v_cache))]
    args = _lib.CacheFp8Args(_ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache), _ints(what, "page_table", page_table, (b, page_table.shape[1]), device),
                             _ints(what, "lengths", lengths, (b,), device), **{name: _ints(what, "tokens" if name == "list" else name, x, shape, device) for name, (x, shape) in lists.items()})
    if b == 0 or entries == 0 or g == 0:
        return
    args.k_stride, args.v_stride, args.k_cache_stride, args.v_cache_stride = *wide, *cache
    args.page_table_stride, args.list_stride = page_table.stride(0), lists["list"][0].stride(0) if lists.get("list", (None,))[0] is not None else 0
    args.batch, args.tokens, args.entries, args.kv_heads, args.head_dim = b, t, entries, g, d
    args.pages, args.page_size, args.max_pages, args.type = pages, max(page_size, 1), page_table.shape[1] if pages and page_size else 0, _TYPES[k.dtype]
    with _buffers_lock:
        if device.index not in _status:
            _device_buffers(device)
    rc = function(ctypes.byref(args), ctypes.byref(scales), device.index, _stream_handle(device.index, device), _ptr(_status[device.index]))
    if rc:
        _raise(what, rc)


def write_cache_fp8(k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, *, tokens=None, counts=None):
    """Writes tokens behind the committed ones of each of B sequences, in 8 bits.

    k, v (B, T, G, D): keys and values of new tokens, fp16 or bf16, D 64 or 128, any T; they may be views of one projection's output.
    k_cache, v_cache, k_scales, v_scales: a cache as :func:`make_cache_fp8` makes it (any page size; the values of a head side by side on 16-byte boundaries,
    the other strides as you like).  page_table (B, P) int32: the pages of each sequence in order; lengths (B,) int32: its committed tokens, not changed here.
    Without ``tokens`` token i is written to place ``lengths[b] + i``; with ``tokens`` (B, A) int32, token ``tokens[b, i]`` is, or nothing where that is
    negative.  ``counts`` (B,) int32: only the first ``counts[b]`` of them.  ``accepted`` and ``counts`` of :func:`verify_drafts` are such tensors.

    Each head of a token gets the least power of two with which its largest finite magnitude stays within 448 (exponents -15..8 for fp16,
    -40..120 for bf16; at the highest, magnitudes end at 240 times it, so that what is read back is finite); its values are divided by it and
    rounded to E4M3, infinities and NaN become NaN.  What has no place - behind the page table, in a page that does not exist, a token number from T on - is
    not written and reported by :func:`device_status` (4).  No two entries of a call may go to the same place of a page.
    At most 65536 heads; steps from token to token, page to page and slot to slot stay below 2^32 elements, the others are free.
    """
    what = "write_cache_fp8"
    # plain CUDA tensors that pass every check: one call into native code; anything else takes the general path below
    rc = _call.write_cache_fp8(k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, tokens, counts)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise(what, rc)
    b, t = k.shape[:2] if k.dim() == 4 else (0, 0)
    entries = t
    if tokens is not None:
        if tokens.dim() != 2:
            raise RuntimeError(f"{what}: tokens must be int32 of shape (B, A)")
        entries = tokens.shape[1]
    _move(what, lib.fp6m_write_cache_fp8, k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, "cache", entries, list=(tokens, (b, entries)), counts=(counts, (b,)))


def read_cache_fp8(k_cache, v_cache, k_scales, v_scales, page_table, lengths, k, v, *, starts=None):
    """Reads tokens of each of B sequences back from a cache that :func:`write_cache_fp8` wrote.

    k, v (B, R, G, D), fp16 or bf16, the type that was written: row i of sequence b becomes token ``starts[b] + i`` (``starts`` (B,) int32, default 0), each
    value times its head's power of two.  Rows of tokens that the sequence does not have - before 0, from ``lengths[b]`` on - are left as they were, and so
    are those in a page that does not exist, which :func:`device_status` reports (4).  The other arguments as in :func:`write_cache_fp8`.
    """
    what = "read_cache_fp8"
    rc = _call.read_cache_fp8(k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, starts)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise(what, rc)
    _move(what, lib.fp6m_read_cache_fp8, k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, "rows",
          k.shape[1] if k.dim() == 4 else 0, starts=(starts, (k.shape[0],) if k.dim() else ()))


def tree_attention_fp8(q, k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, tree, out, *, scale=None):
    """:func:`tree_attention` over a cache in 8 bits (see :func:`make_cache_fp8`): attention of T (at most 64) drafted tokens, or one, of each of B sequences.

    q, k, v, out, page_table, lengths, tree and ``scale`` are as there, with the drafted tokens' queries, keys and values in fp16 or bf16; k_cache,
    v_cache, k_scales and v_scales hold the committed tokens, whose keys and values are the E4M3 values times their powers of two.  Scores, maxima and sums are
    fp32.  The weights of the softmax, each times its value's power of two, are rounded once before they meet the values, and the result once more.

    Up to 32 rows (tokens times heads) per head of keys this takes less time than :func:`tree_attention` over a 16-bit cache, with more rows it takes more (by a fifth to a half) and
    what an 8-bit cache saves is memory.  Up to 32 rows the weights are rounded to fp16, and any E4M3 values will do, with exponent bytes of keys from 0 to 254 and of values from 73 to 247
    (-54 to 120, which holds all that write_cache_fp8 stores).
    With more rows keys and values are widened to the type of q, and the weights rounded to it: the cache must have been written from that type, by :func:`write_cache_fp8` or
    with its exponents and largest values; powers of two that fp16 does
    not hold (exponents below -24 or above 15) are reported by :func:`device_status` (4) where q is that, and results are wrong.  Steps from page to page and slot to slot of k_scales and v_scales stay below 2^32.
    """
    what = "tree_attention_fp8"
    rc = _call.tree_attention_fp8(q, k, v, k_cache, v_cache, page_table, lengths, tree, out, scale, k_scales, v_scales)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise(what, rc)
    args = _tree_args(what, q, k, v, k_cache, v_cache, page_table, lengths, tree, out, scale, torch.float8_e4m3fn)
    device = q.device
    scales = _scales(what, k_scales, v_scales, (*k_cache.shape[:2], k.shape[2]), device)
    if args is None:
        return
    stream = _stream_handle(device.index, device)
    scratch, status = _operator_buffers(what, device, lib.fp6m_tree_attention_fp8_scratch_bytes(_sms(device)), stream)
    rc = lib.fp6m_tree_attention_fp8(ctypes.byref(args), ctypes.byref(scales), _ptr(scratch), scratch.numel(), device.index, stream, _ptr(status))
    if rc:
        _raise(what, rc)


def verify_drafts(target, drafted, tree, uniforms, accepted, counts, next_tokens, *, draft=None):
    """Decides for each of B sequences which of T (at most 64) drafted tokens are accepted, and which token follows them, so that
    the tokens are distributed as the target's probabilities say: with ``draft``, where the children of a token were drawn from it independently of one another, so that an id may
    come twice (for children drawn without repetition the rule is biased); without ``draft``, however they were chosen, as long as it was without looking at ``uniforms``.

    target (B, T, V), fp32, fp16 or bf16: row i holds the target's probabilities of the token after drafted token i.  drafted (B, T) int64: the tokens' ids.
    tree (B, T) or (T,) int64: the masks that :func:`tree_attention` takes; a token's parent is the last earlier one that it sees.
    Token 0 is the token that the step before has chosen and is accepted as it is; where its mask is 0 the sequence is padding (nothing is accepted, the next token is -1).
    uniforms (B, T) float32, 0 <= u < 1: ``uniforms[b, 0]`` draws the next token, the others decide about their drafted token.  draft (B, T, V), like target: the
    probabilities that the children of token i were drawn from; without it they were chosen, not drawn.

    From a token n that is accepted on, with ``r = target[b, n]`` and ``q = draft[b, n]``, its children c are looked at in order: c is accepted, and n goes to c, if
    ``uniforms[b, c] * q[id] < r[id]``; otherwise ``r`` becomes ``max(r - q, 0)`` divided by its sum.  Where none is accepted the next token
    is the lowest x with ``r[0] + ... + r[x] > uniforms[b, 0] * sum(r)``.  Without draft 1 stands for ``q[id]``, and ``r[id]`` becomes 0 in place of the
    subtraction.  Where nothing of r remains, further children are not accepted and the next token is drawn from ``target[b, n]``.  With T = 1 a
    token is drawn from ``target[:, 0]``.  Probabilities that are negative, infinite or NaN count as 0 (-1 is the next token of a row without any), ids outside
    the vocabulary have none; sums are taken in 64 bits.

    Overwritten: accepted (B, T) int32, the accepted tokens' numbers in order, then -1; counts (B,) int32, how many; next_tokens (B,) int64.
    """
    what = "verify_drafts"
    rc = _call.verify_drafts(target, draft, drafted, tree, uniforms, accepted, counts, next_tokens)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise(what, rc)
    if not target.is_cuda:
        raise RuntimeError(f"fp6_marlin_b200.{what} needs CUDA tensors: there is no CPU implementation")
    if target.dtype not in _PROBABILITIES or target.dim() != 3:
        raise RuntimeError(f"{what}: target must be (B, T, V) of float32, float16 or bfloat16")
    b, t, vocab = target.shape
    if t > 64:
        raise RuntimeError(f"{what}: at most 64 drafted tokens")
    device = target.device
    for name, x, dtype, shapes in (("draft", draft, target.dtype, ((b, t, vocab),)), ("drafted", drafted, torch.int64, ((b, t),)), ("tree", tree, torch.int64, ((t,), (b, t))),
                                   ("uniforms", uniforms, torch.float32, ((b, t),)), ("accepted", accepted, torch.int32, ((b, t),)),
                                   ("counts", counts, torch.int32, ((b,),)), ("next_tokens", next_tokens, torch.int64, ((b,),))):
        if x is None and name == "draft":
            continue
        if x.dtype != dtype or tuple(x.shape) not in shapes:
            raise RuntimeError(f"{what}: {name} must be {str(dtype).removeprefix('torch.')} of shape {' or '.join(map(str, shapes))}")
        if x.device != device:
            raise RuntimeError(f"{what}: {name} must be on the same CUDA device as the other tensors")
        if name not in ("draft", "tree") and not x.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be contiguous")
    if vocab > 1 and t and b and (target.stride(2) != 1 or (draft is not None and draft.stride(2) != 1)) or (t > 1 and tree.stride(-1) != 1):
        raise RuntimeError(f"{what}: the rows of target, draft and tree must be contiguous")
    if b == 0 or t == 0:
        return
    if vocab == 0:
        raise RuntimeError(f"{what}: there must be a vocabulary")
    args = _lib.VerifyDraftsArgs(_ptr(target), 0 if draft is None else _ptr(draft), _ptr(drafted), _ptr(tree), _ptr(uniforms), _ptr(accepted), _ptr(counts), _ptr(next_tokens),
                                 (ctypes.c_longlong * 2)(*target.stride()[:2]), (ctypes.c_longlong * 2)(*(target if draft is None else draft).stride()[:2]),
                                 tree.stride(0) if tree.dim() == 2 else 0, b, t, vocab, _PROBABILITIES[target.dtype])
    rc = lib.fp6m_verify_drafts(ctypes.byref(args), device.index, _stream_handle(device.index, device))
    if rc:
        _raise(what, rc)
