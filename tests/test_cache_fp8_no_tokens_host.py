"""Only writing goes without the addresses of keys and values, where there are no tokens: reading writes to them."""
from fp6_marlin_b200 import _lib

ONE = 16                                                            # a non-null, aligned "address"


def test_rows_are_needed_where_they_are_written():
    scales = _lib.CacheScales(ONE, ONE)
    for rows in ((0, ONE), (ONE, 0), (0, 0), (8, ONE)):
        for tokens in (0, 1):
            args = _lib.CacheFp8Args(*rows, *([ONE] * 4), batch=1, tokens=tokens, entries=1, kv_heads=2, head_dim=64, pages=1, page_size=16, max_pages=1)
            assert _lib.lib.fp6m_read_cache_fp8(args, scales, 0, None, None) == _lib.ERR_BAD_ARG
            if tokens:
                assert _lib.lib.fp6m_write_cache_fp8(args, scales, 0, None, None) == _lib.ERR_BAD_ARG
