"""What of the 8-bit cache, attention over it and the verification of drafted tokens runs without a GPU: the empty cache, refusals."""
import ctypes

import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200 import _lib

ONE = 16                                                            # a non-null, aligned "address"


def test_an_empty_cache():
    k, v, ks, vs = fm.make_cache_fp8(5, 24, 3, 64, device="cpu")
    assert k.shape == v.shape == (5, 24, 3, 64) and k.dtype == v.dtype == torch.float8_e4m3fn and not k.view(torch.uint8).any()
    assert ks.shape == vs.shape == (5, 24, 3) and ks.dtype == torch.uint8 and ks.stride() == (72, 1, 24) and (vs == 127).all()


def test_there_is_no_cpu_path():
    z = torch.zeros((1, 1, 1, 64), dtype=torch.float16)
    cache, table, lengths = fm.make_cache_fp8(1, 16, 1, 64, device="cpu"), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        fm.write_cache_fp8(z, z, *cache, table, lengths)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        fm.read_cache_fp8(*cache, table, lengths, z, z)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        fm.tree_attention_fp8(z, z, z, *cache, table, lengths, torch.ones(1, dtype=torch.int64), z)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        fm.verify_drafts(torch.ones((1, 1, 8)), torch.zeros((1, 1), dtype=torch.int64), torch.ones(1, dtype=torch.int64), torch.zeros((1, 1)), table, lengths, torch.zeros(1, dtype=torch.int64))


def _changed(args, change):
    copy = type(args).from_buffer_copy(args)
    for name, value in change.items():
        setattr(copy, name, value)
    return copy


@pytest.mark.parametrize("function", ["fp6m_write_cache_fp8", "fp6m_read_cache_fp8"])
def test_cache_entries_refuse_before_they_touch_the_gpu(function):
    args = _lib.CacheFp8Args(*([ONE] * 6), batch=1, tokens=1, entries=1, kv_heads=2, head_dim=64, pages=1, page_size=16, max_pages=1)
    scales = _lib.CacheScales(ONE, ONE)
    call = lambda s=scales, **change: getattr(_lib.lib, function)(_changed(args, change), s, 0, None, None)     # noqa: E731
    three = ctypes.c_longlong * 3
    assert call(batch=-1) == call(entries=-1) == call(tokens=-2) == call(type=2) == call(type=-1) == _lib.ERR_BAD_ARG
    assert call(head_dim=96) == call(page_size=0) == call(kv_heads=-1) == call(kv_heads=(1 << 16) + 1) == call(pages=-1) == call(max_pages=-1) == _lib.ERR_PROB_SHAPE
    assert call(k=0) == call(v=24) == call(lengths=0) == call(k_cache=8) == call(v_cache=0) == call(page_table=0) == call(list_stride=-1) == call(page_table_stride=-1) == _lib.ERR_BAD_ARG
    assert call(k_stride=three(0, 4, 0)) == call(v_stride=three(-8, 0, 0)) == call(k_cache_stride=three(0, 8, 0)) == call(v_cache_stride=three(0, 0, -16)) == _lib.ERR_BAD_ARG
    assert call(_lib.CacheScales(0, ONE)) == call(_lib.CacheScales(ONE, ONE, three(0, 0, -1))) == call(None) == getattr(_lib.lib, function)(None, scales, 0, None, None) == _lib.ERR_BAD_ARG
    for page_size, max_pages in ((64, (1 << 25) - 32), (1, (1 << 31) - 256), (1 << 30, 2)):
        assert call(page_size=page_size, max_pages=max_pages) == _lib.ERR_PROB_SHAPE
    far = 1 << 32
    assert call(k_stride=three(0, far, 0)) == call(v_stride=three(0, far, 0)) == call(k_cache_stride=three(far, 0, 0)) == call(v_cache_stride=three(0, far, 0)) == _lib.ERR_PROB_SHAPE
    assert call(_lib.CacheScales(ONE, ONE, three(far, 0, 0))) == call(_lib.CacheScales(ONE, ONE, three(), three(0, far, 0))) == _lib.ERR_PROB_SHAPE
    assert call(batch=0) == call(entries=0) == call(kv_heads=0) == _lib.OK


def test_attention_refuses_before_it_touches_the_gpu():
    args, scales = _lib.TreeAttentionArgs(*([ONE] * 9), batch=1, tokens=1, heads=2, kv_heads=2, head_dim=64, pages=1, page_size=16, max_pages=1), _lib.CacheScales(ONE, ONE)
    call = lambda s=scales, **change: _lib.lib.fp6m_tree_attention_fp8(_changed(args, change), s, ONE, 1 << 30, 0, None, None)     # noqa: E731
    three = ctypes.c_longlong * 3
    assert call(tokens=65) == call(head_dim=80) == call(kv_heads=3) == call(page_size=0) == call(heads=3, kv_heads=2) == _lib.ERR_PROB_SHAPE
    assert call(batch=-1) == call(type=2) == call(q=0) == call(out=24) == call(page_table=0) == call(lengths=0) == call(tree=0) == _lib.ERR_BAD_ARG
    assert call(k_cache_stride=three(0, 8, 0)) == call(v_cache_stride=three(24, 0, 0)) == call(q_stride=three(0, 0, 4)) == _lib.ERR_BAD_ARG      # 16 values of 8 bits, 8 of 16
    assert call(_lib.CacheScales(ONE, 0)) == call(_lib.CacheScales(ONE, ONE, three(), three(-1, 0, 0))) == call(None) == _lib.ERR_BAD_ARG
    far = 1 << 32
    assert call(_lib.CacheScales(ONE, ONE, three(far, 0, 0))) == call(_lib.CacheScales(ONE, ONE, three(), three(0, far, 0))) == _lib.ERR_PROB_SHAPE
    assert call(batch=0) == call(tokens=0) == call(heads=0) == _lib.OK
    for page_size, max_pages in ((64, (1 << 25) - 32), (1, (1 << 31) - 256), (1 << 30, 2)):
        assert call(page_size=page_size, max_pages=max_pages, tokens=64) == _lib.ERR_PROB_SHAPE


def test_verification_refuses_before_it_touches_the_gpu():
    args = _lib.VerifyDraftsArgs(ONE, 0, *([ONE] * 6), batch=1, tokens=1, vocab=8, type=_lib.TYPE_F32)
    call = lambda **change: _lib.lib.fp6m_verify_drafts(_changed(args, change), 0, None)     # noqa: E731
    two = ctypes.c_longlong * 2
    assert call(batch=-1) == call(tokens=-1) == call(vocab=-1) == call(type=3) == call(type=-1) == _lib.ERR_BAD_ARG
    assert call(tokens=65) == call(vocab=0) == call(vocab=(1 << 30) + 1) == call(batch=1 << 30) == _lib.ERR_PROB_SHAPE
    assert call(target=0) == call(target=18) == call(draft=18) == call(target=17, type=_lib.TYPE_F16) == call(drafted=0) == call(tree=0) == call(uniforms=0) == _lib.ERR_BAD_ARG
    assert call(accepted=0) == call(counts=0) == call(next_tokens=0) == call(tree_stride=-1) == call(target_stride=two(0, -1)) == call(draft=ONE, draft_stride=two(-1, 0)) == _lib.ERR_BAD_ARG
    assert _lib.lib.fp6m_verify_drafts(None, 0, None) == _lib.ERR_BAD_ARG
    assert call(batch=0) == call(tokens=0) == call(batch=0, vocab=0) == _lib.OK
