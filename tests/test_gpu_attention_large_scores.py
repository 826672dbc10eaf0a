"""Attention whose scores are far larger than 2^24, over caches in 16 and in 8 bits: rows whose largest score stands out from the others attend to that token alone.

A score is off by at most slack = D * 2^-23 * scale * sum |q k|, its product with log2(e) by 2^-24 of it: where the largest leads by four times the slack, and by 40 beside, the other weights are below 2^-40
(no more than 64 * 2^-40 of the values in all).  The weight of the largest is rounded once, the result once more: 4 u = 2^-9 (fp16), 2^-6 (bf16) with a lot to spare.
"""
import pytest
import torch

import fp6_marlin_b200 as fm
import test_gpu_tree_attention as wide
import test_gpu_tree_attention_fp8 as narrow

pytestmark = pytest.mark.gpu


def _keys_and_values(x, i, n, fp8):
    at = torch.arange(n, device="cuda")
    page = x["k_cache"].shape[1]
    cached = [narrow.tokens(x, name, i, at)[0] if fp8 else x[name + "_cache"][x["page_table"][i].long()[at // page], at % page].double() for name in ("k", "v")]
    return [torch.cat([c, x[name][i].double()]) for c, name in zip(cached, ("k", "v"))]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,h,g,d", [(1, 4, 1, 128), (6, 8, 2, 128), (12, 4, 1, 128), (20, 8, 2, 64), (64, 8, 2, 128), (40, 32, 4, 64)])
@pytest.mark.parametrize("scale", [2.0 ** 20, 2.0 ** 26, -2.0 ** 30, 2.0 ** 60, 2.0 ** 100])
def test_the_largest_score_takes_all(t, h, g, d, scale, dtype, fp8):
    lengths = [300, 5000]
    x = narrow.inputs(2, t, h, g, d, lengths, 16, dtype) if fp8 else wide._inputs(2, t, h, g, d, lengths, 16, dtype)
    x["tree"][:] = 1 << torch.arange(t, device="cuda")             # every token sees the cached ones and itself
    out = (narrow.run if fp8 else wide._run)(x, scale=scale).double()
    assert out.isfinite().all() and fm.device_status() == 0
    clear = 0
    for i, n in enumerate(lengths):
        keys, values = (v.repeat_interleave(h // g, 1) for v in _keys_and_values(x, i, n, fp8))
        for j in range(t):
            at = [*range(n), n + j]
            q = x["q"][i, j].double()
            s, size = torch.einsum("hd,nhd->hn", q, keys[at]) * scale, torch.einsum("hd,nhd->hn", q.abs(), keys[at].abs()) * abs(scale)
            top, second = s.topk(2, 1).values.T
            lead = top - second > 4 * d * 2.0 ** -23 * size.amax(1) + 40
            expect = values[at][s.argmax(1), torch.arange(h, device="cuda")]
            u = 4 * narrow.BITS[dtype]
            most = values[at].abs().amax((0, 2))[:, None]
            assert ((out[i, j] - expect).abs() <= u * expect.abs() + 2.0 ** -34 * most + 2.0 ** -24)[lead].all()
            clear += int(lead.sum())
    assert clear >= t * h                                          # (half of the rows at least)
