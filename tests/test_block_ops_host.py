"""What of the operators between the products runs without a GPU: the masks of a tree, 8-bit weights, refusals."""
import pytest
import torch

import fp6_marlin_b200 as fm
from fp6_marlin_b200 import _lib


def test_tree_masks():
    #      0   1 hangs on 0   2 on 0   3 on 1   4 beside 0   5 padding
    masks = fm.tree_masks(torch.tensor([-1, 0, 0, 1, -1, -2]))
    assert masks.tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0]
    chain = fm.tree_masks(torch.arange(64) - 1)
    assert [int(m) & (1 << 64) - 1 for m in chain] == [(2 << i) - 1 for i in range(64)]
    two = fm.tree_masks(torch.tensor([[-1, 0], [-1, -1]]))
    assert two.tolist() == [[1, 3], [1, 2]]
    for bad in (torch.arange(65) - 1, torch.tensor([0]), torch.tensor([-3]), torch.tensor([-1, 1])):
        with pytest.raises(ValueError):
            fm.tree_masks(bad)


@pytest.mark.parametrize("n,k", [(8, 16), (128, 128), (136, 272), (300, 1040)])
def test_fp8_weight(n, k):
    w = torch.randn((n, k), generator=torch.Generator().manual_seed(n)) * 0.02
    w[: n // 2, : min(k, 128)] = 0
    q, s = fm.make_fp8_weight(w)
    assert q.shape == (n, k) and s.shape == (-(-n // 128), -(-k // 128)) and (s > 0).all()
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            block = w[128 * i:128 * i + 128, 128 * j:128 * j + 128].double()
            assert abs(float(s[i, j]) - max(float(block.abs().max()), 1e-30) / 448) <= 2.0 ** -22 * float(s[i, j])
            back = q[128 * i:128 * i + 128, 128 * j:128 * j + 128].double() * float(s[i, j])
            assert ((back - block).abs() <= (block.abs() * 2.0 ** -4).clamp(min=float(s[i, j]) * 2.0 ** -10) * (1 + 2.0 ** -10)).all()
    with pytest.raises(ValueError):
        fm.make_fp8_weight(w[0])


def test_there_is_no_cpu_path():
    x = torch.zeros((2, 128), dtype=torch.float16)
    q = torch.zeros((2, 128)).to(torch.float8_e4m3fn)
    s = torch.ones((2, 1))
    with pytest.raises(RuntimeError):
        fm.rms_norm(x, x[0], x.clone())
    with pytest.raises(RuntimeError):
        fm.quantize_fp8(x, q, s)
    with pytest.raises(RuntimeError):
        fm.mul_fp8(q, q, x[:, :2], s, s)
    z = torch.zeros((1, 1, 1, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError):
        fm.tree_attention(z, z, z, z, z, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int64), z)


def test_c_entries_refuse_before_they_touch_the_gpu():
    lib, one = _lib.lib, 16                                         # a non-null, aligned "address"
    assert lib.fp6m_rms_norm(one, one, 0, 0, one, 0, 1, 12, 1e-6, 0, 0, None) == _lib.ERR_BAD_ARG          # no multiple of 8
    assert lib.fp6m_rms_norm(one, one, one, 0, one, 0, 1, 8, 1e-6, 0, 0, None) == _lib.ERR_BAD_ARG         # a residual without a place for the sum
    assert lib.fp6m_rms_norm(one, 0, 0, 0, one, 0, 1, 8, 1e-6, 0, 0, None) == _lib.ERR_BAD_ARG
    assert lib.fp6m_rms_norm(one, one, 0, 0, one + 2, 0, 1, 8, 1e-6, 0, 0, None) == _lib.ERR_BAD_ARG
    assert lib.fp6m_rms_norm(one, one, 0, 0, one, 0, 1, 8, 1e-6, 2, 0, None) == _lib.ERR_BAD_ARG
    assert lib.fp6m_rms_norm(0, 0, 0, 0, 0, 0, 0, 8, 1e-6, 0, 0, None) == _lib.OK
    assert lib.fp6m_quantize_fp8(one, one, 0, 1, 8, 0, 0, None) == _lib.ERR_BAD_ARG
    mul = lambda m, n, k, a=one, c=one, kind=0: lib.fp6m_mul_fp8(a, one, c, one, one, m, n, k, kind, one, 1 << 30, 0, None, 0)     # noqa: E731
    assert mul(1, 8, 24) == _lib.ERR_PROB_SHAPE and mul(1, 12, 16) == _lib.ERR_PROB_SHAPE and mul(-1, 8, 16) == _lib.ERR_BAD_ARG
    assert mul(1, 8, 16, kind=7) == _lib.ERR_BAD_ARG and mul(1, 8, 16, a=0) == _lib.ERR_BAD_ARG and mul(1, 8, 16, c=24) == _lib.ERR_BAD_ARG
    assert mul(0, 8, 16) == _lib.OK and mul(1, 0, 16) == _lib.OK
    args = _lib.TreeAttentionArgs(*([one] * 9), batch=1, tokens=1, heads=2, kv_heads=2, head_dim=64, pages=1, page_size=16, max_pages=1)
    tree = lambda **change: lib.fp6m_tree_attention(_changed(args, change), one, 1 << 30, 0, None, 0)     # noqa: E731
    assert tree(tokens=65) == _lib.ERR_PROB_SHAPE and tree(head_dim=80) == _lib.ERR_PROB_SHAPE and tree(kv_heads=3) == _lib.ERR_PROB_SHAPE
    assert tree(page_size=0) == _lib.ERR_PROB_SHAPE and tree(batch=-1) == _lib.ERR_BAD_ARG and tree(type=5) == _lib.ERR_BAD_ARG and tree(q=0) == _lib.ERR_BAD_ARG
    assert tree(out=24) == _lib.ERR_BAD_ARG and tree(page_table=0) == _lib.ERR_BAD_ARG and tree(batch=0) == _lib.OK
    assert lib.fp6m_tree_attention(None, one, 1 << 30, 0, None, 0) == _lib.ERR_BAD_ARG


def _changed(args, change):
    copy = type(args).from_buffer_copy(args)
    for name, value in change.items():
        setattr(copy, name, value)
    return copy


def test_products_whose_places_do_not_fit_an_int():
    lib, one = _lib.lib, 16
    for m, n, k in ((1, 8, (1 << 31) - 128), (100, 8, (1 << 31) - 16), (1, (1 << 31) - 128, 16), ((1 << 31) - 200, 8, 16)):
        assert lib.fp6m_mul_fp8(one, one, one, one, one, m, n, k, 0, one, 1 << 40, 0, None, 0) == _lib.ERR_PROB_SHAPE
        assert lib.fp6m_mul_fp8_scratch_bytes(m, n, k, 148) == 256


def test_tables_whose_tokens_do_not_fit_an_int():
    """2^31 - 2048 of them and more: the look-up of pages goes up to 4160 tokens past a sequence's end."""
    args = _lib.TreeAttentionArgs(*([16] * 9), batch=1, tokens=64, heads=2, kv_heads=1, head_dim=64, pages=1)
    for page_size, max_pages in ((64, (1 << 25) - 32), (1, (1 << 31) - 256), (1 << 30, 2)):
        assert _lib.lib.fp6m_tree_attention(_changed(args, dict(page_size=page_size, max_pages=max_pages)), 16, 1 << 40, 0, None, 0) == _lib.ERR_PROB_SHAPE
