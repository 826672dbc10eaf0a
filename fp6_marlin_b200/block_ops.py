"""What stands between the weight products of a decoder block: norm, rounding to 8 bits, the 8-bit product, attention.

``rms_norm`` and ``quantize_fp8`` make the rows that ``mul`` (16 bits) and ``mul_fp8`` (E4M3 with a scale for each 128
neighbours) take; ``mul_fp8`` multiplies them by a weight kept in 8 bits, for layers that lose too much in INT4 / FP6;
``tree_attention`` lets a tree of drafted tokens, or a single next token, attend to a paged cache.  As with ``mul`` the outputs
are tensors of the caller that are overwritten, all calls run asynchronously on the current stream of their device, and
PyTorch is used for memory, streams and device management only.  The reference has no counterpart of these; its layer lists
(bench.py:53-86) name the products on either side.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .api import _buffers_lock, _call, _device_buffers, _ptr, _sm_count, _status, _stream_handle, _zeros
from ._lib import lib

GROUP = 128                                       # neighbours that share a scale
E4M3_MAX = 448.0
SMALLEST = 1e-30                                  # largest magnitude that a group of zeros is given
_TYPES = {torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}

_call.bind_operators(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
    "fp6m_rms_norm", "fp6m_quantize_fp8", "fp6m_mul_fp8", "fp6m_mul_fp8_scratch_bytes", "fp6m_tree_attention", "fp6m_tree_attention_scratch_bytes")))
_OWNERS = {"mul_fp8": 1, "tree_attention": 2}     # of a scratch, as the native call path numbers them

_scratch: dict[tuple, list[torch.Tensor]] = {}    # (operator, device, stream) -> buffers, the last is in use


def _operator_buffers(name: str, device: torch.device, nbytes: int, stream: int):
    """Scratch and status word of an operator on one stream: as for the GEMMs a buffer is zeroed once, and one that a larger
    one replaces is kept, because a call of another thread or a captured graph may hold its address."""
    key = (name, device.index, stream)
    with _buffers_lock:
        if device.index not in _status:
            _device_buffers(device)
        buffers = _scratch.setdefault(key, [])
        if not buffers or buffers[-1].numel() < nbytes:
            if buffers:
                nbytes = max(nbytes, 2 * buffers[-1].numel())
            buffers.append(_zeros(nbytes, device))
            _call.set_operator_scratch(_OWNERS[name], device.index, stream, _ptr(buffers[-1]), nbytes)
        return buffers[-1], _status[device.index]


def _sms(device: torch.device) -> int:
    if device.index not in _sm_count:
        _sm_count[device.index] = torch.cuda.get_device_properties(device.index).multi_processor_count
    return _sm_count[device.index]


def _check(what: str, device: torch.device, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise RuntimeError(f"{what}: {name} must be on the same CUDA device as the other tensors")
        if not t.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be contiguous")


def _raise(what: str, rc: int):
    if rc == _lib.ERR_PROB_SHAPE:
        raise RuntimeError(f"{what}: the shape is not supported")
    if rc == _lib.ERR_BAD_ARG:                     # (what else it stands for is checked before)
        raise RuntimeError(f"{what}: the tensors must start on 16-byte boundaries")
    if rc == _lib.ERR_CUDA:
        raise RuntimeError(f"{what}: CUDA error: {_lib.last_cuda_error()}")
    raise RuntimeError(f"{what} failed with code {rc}")


def _rows(what, x, y, scales):
    """Checks what the two row operators have in common; returns (M, N)."""
    if not x.is_cuda:
        raise RuntimeError(f"fp6_marlin_b200.{what} needs CUDA tensors: there is no CPU implementation")
    if x.dtype not in _TYPES or x.dim() != 2:
        raise RuntimeError(f"{what}: x must be a matrix of float16 or bfloat16")
    m, n = x.shape
    if n % 8:
        raise RuntimeError(f"{what}: rows must have a multiple of 8 values, got {n}")
    if y.shape != x.shape or y.dtype != (x.dtype if scales is None else torch.float8_e4m3fn):
        raise RuntimeError(f"{what}: the output must have x's shape, and x's type, or float8_e4m3fn where there are scales")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (m, -(-n // GROUP))):
        raise RuntimeError(f"{what}: scales must be float32 of shape ({m}, {-(-n // GROUP)})")
    return m, n


def rms_norm(x, weight, y, eps=1e-6, *, scales=None, residual=None, residual_out=None):
    """``h = x + residual``, ``y = h * rsqrt(mean(h**2) + eps) * weight`` for the rows of ``x`` (M, N), fp16 or bf16.

    ``residual`` (optional, like x) is added in fp32; the sum, rounded once, goes to ``residual_out`` (default: ``residual``
    itself, in place), and the norm goes on with the sum before that rounding.  Without ``scales`` ``y`` has x's type; with ``scales``
    (M, ceil(N/128)) float32, ``y`` is float8_e4m3fn, the result divided by its scale (one for each 128 neighbours of a row: their
    largest magnitude / 448), and ``y * scales`` stands for the result: what :func:`mul_fp8` takes.  N must be a multiple of 8.
    """
    # plain CUDA tensors that pass every check: one call into native code; anything else takes the general path below
    rc = _call.rms_norm(x, weight, y, eps, scales, residual, residual_out)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise("rms_norm", rc)
    m, n = _rows("rms_norm", x, y, scales)
    if weight.dtype != x.dtype or weight.shape != (n,):
        raise RuntimeError(f"rms_norm: weight must hold {n} values of x's type")
    if residual is None:
        if residual_out is not None:
            raise RuntimeError("rms_norm: residual_out needs a residual")
    else:
        if residual_out is None:
            residual_out = residual
        for t in (residual, residual_out):
            if t.dtype != x.dtype or t.shape != x.shape:
                raise RuntimeError("rms_norm: residual and residual_out must have x's shape and type")
    device = x.device
    _check("rms_norm", device, x=x, weight=weight, y=y, scales=scales, residual=residual, residual_out=residual_out)
    rc = lib.fp6m_rms_norm(_ptr(x), _ptr(weight), 0 if residual is None else _ptr(residual), 0 if residual is None else _ptr(residual_out), _ptr(y),
                           0 if scales is None else _ptr(scales), m, n, eps, _TYPES[x.dtype], device.index, _stream_handle(device.index, device))
    if rc:
        _raise("rms_norm", rc)


def quantize_fp8(x, q, scales):
    """Rounds the rows of ``x`` (M, N), fp16 or bf16, to E4M3: ``scales[m, g]`` (float32) is the largest magnitude of 128
    neighbours / 448 and ``q`` (float8_e4m3fn) the values divided by it.  N must be a multiple of 8."""
    if scales is None:
        raise RuntimeError("quantize_fp8: scales are needed")
    rc = _call.quantize_fp8(x, q, scales)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise("quantize_fp8", rc)
    m, n = _rows("quantize_fp8", x, q, scales)
    device = x.device
    _check("quantize_fp8", device, x=x, q=q, scales=scales)
    rc = lib.fp6m_quantize_fp8(_ptr(x), _ptr(q), _ptr(scales), m, n, _TYPES[x.dtype], device.index, _stream_handle(device.index, device))
    if rc:
        _raise("quantize_fp8", rc)


def make_fp8_weight(w):
    """``w`` (N, K), any floating type -> (float8_e4m3fn of the same shape, float32 scales (ceil(N/128), ceil(K/128))): each block of
    128 x 128 values is divided by its largest magnitude / 448.  On w's device, with torch's operations (done once per layer)."""
    if w.dim() != 2 or not w.is_floating_point():
        raise ValueError("make_fp8_weight: expected a matrix of floating-point values")
    n, k = w.shape
    nb, kb = -(-n // GROUP), -(-k // GROUP)
    q = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=w.device)
    s = torch.empty((nb, kb), dtype=torch.float32, device=w.device)
    for b in range(nb):
        rows = w.detach()[b * GROUP:(b + 1) * GROUP].float()
        wide = torch.nn.functional.pad(rows, (0, kb * GROUP - k)).view(rows.shape[0], kb, GROUP)
        s[b] = wide.abs().amax((0, 2)).clamp(min=SMALLEST) / E4M3_MAX
        q[b * GROUP:(b + 1) * GROUP] = (wide / s[b][:, None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows.shape[0], -1)[:, :k].to(torch.float8_e4m3fn)
    return q, s


def mul_fp8(A, B, C, sa, sb):
    """``C[M, N] = (A * sa) @ (B * sb).T`` with A (M, K) and B (N, K) in float8_e4m3fn, C fp16 or bf16, overwritten.

    ``sa`` (M, ceil(K/128)) float32 holds a scale for each 128 neighbours of a row of A, ``sb`` (ceil(N/128), ceil(K/128)) one for
    each 128 x 128 block of B.  Sums are fp32 and rounded once.  K must be a multiple of 16 and N of 8."""
    rc = _call.mul_fp8(A, B, C, sa, sb)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise("mul_fp8", rc)
    if not A.is_cuda:
        raise RuntimeError("fp6_marlin_b200.mul_fp8 needs CUDA tensors: there is no CPU implementation")
    if A.dtype != torch.float8_e4m3fn or B.dtype != torch.float8_e4m3fn or A.dim() != 2 or B.dim() != 2:
        raise RuntimeError("mul_fp8: A and B must be matrices of float8_e4m3fn")
    m, k = A.shape
    n = B.shape[0]
    if B.shape[1] != k or C.shape != (m, n):
        raise RuntimeError("mul_fp8: A (M, K), B (N, K) and C (M, N) do not fit together")
    if C.dtype not in _TYPES:
        raise RuntimeError("mul_fp8: C must be float16 or bfloat16")
    if k % 16 or n % 8:
        raise RuntimeError(f"mul_fp8: K must be a multiple of 16 and N of 8, got {k} and {n}")
    blocks = -(-k // GROUP)
    if sa.dtype != torch.float32 or sb.dtype != torch.float32 or sa.shape != (m, blocks) or sb.shape != (-(-n // GROUP), blocks):
        raise RuntimeError(f"mul_fp8: sa must be float32 of shape ({m}, {blocks}) and sb of shape ({-(-n // GROUP)}, {blocks})")
    device = A.device
    _check("mul_fp8", device, A=A, B=B, C=C, sa=sa, sb=sb)
    if m == 0 or n == 0:
        return
    stream = _stream_handle(device.index, device)
    scratch, status = _operator_buffers("mul_fp8", device, lib.fp6m_mul_fp8_scratch_bytes(m, n, k, _sms(device)), stream)
    rc = lib.fp6m_mul_fp8(_ptr(A), _ptr(B), _ptr(C), _ptr(sa), _ptr(sb), m, n, k, _TYPES[C.dtype], _ptr(scratch), scratch.numel(), device.index, stream, _ptr(status))
    if rc:
        _raise("mul_fp8", rc)


def tree_masks(parents):
    """Parents of drafted tokens (..., T) -> the int64 masks that :func:`tree_attention` takes: bit j of mask i is set where
    token j is i itself or one of its ancestors.  ``parents[..., i]`` is an earlier token, -1 for one that hangs on the last
    committed token, or -2 for padding, whose mask is 0."""
    t = parents.shape[-1]
    if t > 64:
        raise ValueError("tree_masks: at most 64 drafted tokens")
    p = parents.long()
    if bool((p >= torch.arange(t, device=p.device)).any()) or bool((p < -2).any()):
        raise ValueError("tree_masks: a parent is an earlier token, -1 or -2")
    masks = torch.zeros_like(p)
    for i in range(t):
        above = masks.gather(-1, p[..., i:i + 1].clamp(min=0))[..., 0]
        own = torch.full_like(above, 1 << i if i < 63 else -(1 << 63))
        masks[..., i] = torch.where(p[..., i] == -2, 0, torch.where(p[..., i] >= 0, above, 0) | own)
    return masks


def _strides(what, name, t, dtype, shape, device, written=False):
    if t.dtype != dtype or t.dim() != 4 or tuple(t.shape) != shape:
        raise RuntimeError(f"{what}: {name} must be of shape {shape} and q's type")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} must be on q's device")
    s = [shape[3] if size == 1 else step for size, step in zip(shape[:3], t.stride())] + [t.stride(3)]      # (that of a single place says nothing)
    if t.numel() and (s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or t.data_ptr() % 16):
        raise RuntimeError(f"{what}: the values of a head of {name} must lie next to one another, on 16-byte boundaries")
    if written and any(size > 1 and step == 0 for size, step in zip(shape, s)):
        raise RuntimeError(f"{what}: places of {name} share memory")
    return (ctypes.c_longlong * 3)(*s[:3])


def tree_attention(q, k, v, k_cache, v_cache, page_table, lengths, tree, out, *, scale=None):
    """Attention of T (at most 64) drafted tokens of each of B sequences over a paged cache and over one another.

    q (B, T, H, D), k and v (B, T, G, D): the drafted tokens' queries, keys and values, fp16 or bf16, D 64 or 128, H a multiple
    of G; they may be views of one projection's output.  k_cache and v_cache (pages, page size, G, D): the cache, any
    page size.  page_table (B, P) int32: the pages of each sequence in order; lengths (B,) int32: its committed tokens.
    tree (B, T) or (T,) int64: bit j of entry i says whether drafted token i sees drafted token j (see :func:`tree_masks`); every
    token sees all committed ones, except that an entry of 0 marks padding, which sees nothing and gives zeros.  Bits from T
    on mean nothing.  With T = 1 and tree = 1 this is ordinary decoding.  out: like q, overwritten.  ``scale`` defaults to ``D ** -0.5``.

    Scores, maxima and sums are fp32; the weights of the softmax are rounded once, to q's type, before they meet the values, the result
    once more.  Lengths and page numbers stay on the device: lengths are cut to what the page table can hold, and a page number that
    does not exist hides its tokens and is reported by :func:`device_status` (4).  What lies behind a sequence's last
    committed token, in the table or in a page, is not read.
    """
    what = "tree_attention"
    rc = _call.tree_attention(q, k, v, k_cache, v_cache, page_table, lengths, tree, out, scale)
    if rc == _lib.OK:
        return
    if rc > 0:
        _raise(what, rc)
    if not q.is_cuda:
        raise RuntimeError("fp6_marlin_b200.tree_attention needs CUDA tensors: there is no CPU implementation")
    if q.dtype not in _TYPES or q.dim() != 4:
        raise RuntimeError(f"{what}: q must be (B, T, H, D) of float16 or bfloat16")
    b, t, h, d = q.shape
    g = k.shape[2] if k.dim() == 4 else 0
    if t > 64 or d not in (64, 128) or g == 0 or h % g:
        raise RuntimeError(f"{what}: at most 64 tokens, heads of 64 or 128 values, and a multiple of the heads of keys as heads of queries")
    if k_cache.dim() != 4 or page_table.dim() != 2:
        raise RuntimeError(f"{what}: the cache must be (pages, page size, {g}, {d}) and the page table (B, P)")
    pages, page_size = k_cache.shape[:2]
    device = q.device
    args = _lib.TreeAttentionArgs(
        _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(k_cache), _ptr(v_cache), _ptr(page_table), _ptr(lengths), _ptr(tree),
        _strides(what, "q", q, q.dtype, (b, t, h, d), device), _strides(what, "k", k, q.dtype, (b, t, g, d), device),
        _strides(what, "v", v, q.dtype, (b, t, g, d), device), _strides(what, "out", out, q.dtype, (b, t, h, d), device, True),
        _strides(what, "k_cache", k_cache, q.dtype, (pages, page_size, g, d), device),
        _strides(what, "v_cache", v_cache, q.dtype, (pages, page_size, g, d), device))
    if page_table.dtype != torch.int32 or page_table.shape[0] != b or lengths.dtype != torch.int32 or lengths.shape != (b,):
        raise RuntimeError(f"{what}: page_table must be int32 (B, P) and lengths int32 (B,)")
    if tree.dtype != torch.int64 or tree.shape not in ((t,), (b, t)):
        raise RuntimeError(f"{what}: tree must be int64 of shape ({t},) or ({b}, {t})")
    if page_table.device != device or lengths.device != device or tree.device != device:
        raise RuntimeError(f"{what}: page_table, lengths and tree must be on q's device")
    if any(x.numel() and x.shape[-1] > 1 and x.stride(-1) != 1 for x in (page_table, lengths, tree)):
        raise RuntimeError(f"{what}: the rows of page_table and tree, and lengths, must be contiguous")
    if b == 0 or t == 0 or h == 0:
        return
    args.page_table_stride, args.tree_stride = page_table.stride(0), tree.stride(0) if tree.dim() == 2 else 0
    args.batch, args.tokens, args.heads, args.kv_heads, args.head_dim = b, t, h, g, d
    args.pages, args.page_size, args.max_pages, args.type = pages, max(page_size, 1), page_table.shape[1] if pages and page_size else 0, _TYPES[q.dtype]
    args.scale = d ** -0.5 if scale is None else scale
    stream = _stream_handle(device.index, device)
    scratch, status = _operator_buffers(what, device, lib.fp6m_tree_attention_scratch_bytes(_sms(device)), stream)
    rc = lib.fp6m_tree_attention(ctypes.byref(args), _ptr(scratch), scratch.numel(), device.index, stream, _ptr(status))
    if rc:
        _raise(what, rc)
