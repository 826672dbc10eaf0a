"""tree_attention_fp8 at the ends of what the types hold: values whose powers of two lie 150 apart, queries near the largest bf16.  Bounds: see test_gpu_tree_attention_fp8.py."""
import pytest
import torch

import fp6_marlin_b200 as fm
from test_gpu_tree_attention_fp8 import SHAPES, _bytes, check, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("lengths", [[900, 70], [5000, 0]])
def test_values_of_zero_beside_very_large_ones(t, h, g, d, lengths):
    """Half of the cached tokens have values of zero, for which write_cache_fp8 stores the lowest exponent, the others values of about 2^100; both count as much in the softmax's sum."""
    x = inputs(2, t, h, g, d, lengths, 16, torch.bfloat16)
    x["v_scales"] += 107
    _bytes(x["v_cache"])[:, ::2], x["v_scales"][:, ::2] = 0, 127 - 40
    check(run(x), x)
    x["v"][:] = 0
    check(run(x), x)
    x["v"][:] = 2.0 ** -100                                        # drafted values that are as small as can be beside them
    check(run(x), x)
    assert fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", SHAPES)
@pytest.mark.parametrize("run_length", [16, 64, 192, 2500])
@pytest.mark.parametrize("zeros_first", [True, False])
def test_runs_of_zeros_and_of_very_large_values(t, h, g, d, run_length, zeros_first):
    """As above, by turns of tokens: a maximum that grows by 2^140 within a warp's tokens, between warps and between multiprocessors leaves the tokens before it in the sum."""
    lengths, page = [5000, 700], 16
    x = inputs(2, t, h, g, d, lengths, page, torch.bfloat16)
    x["v_scales"] += 107
    x["q"] = x["q"] / 16                                           # (so that many tokens count)
    for i, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        at = at[(at // run_length % 2 == 0) == zeros_first]
        rows, slots = x["page_table"][i].long()[at // page], at % page
        _bytes(x["v_cache"])[rows, slots], x["v_scales"][rows, slots] = 0, 127 - 40
    x["v"][:] = 0
    check(run(x), x)


@pytest.mark.parametrize("t,h,g,d", SHAPES)
def test_small_and_large_values_as_write_cache_fp8_writes_them(t, h, g, d):
    """From 2^-60, below what the lowest exponent holds, to 2^110, through the cache itself."""
    x = inputs(2, t, h, g, d, [900, 70], 16, torch.bfloat16)
    pages, page = x["k_cache"].shape[:2]
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn((pages, page, g, d), generator=gen, device="cuda").bfloat16()
    v = (torch.randn((pages, page, g, d), generator=gen, device="cuda") * torch.exp2(torch.randint(-60, 111, (pages, page, g, 1), generator=gen, device="cuda").float())).bfloat16()
    table, none = torch.arange(pages, dtype=torch.int32, device="cuda")[:, None], torch.zeros(pages, dtype=torch.int32, device="cuda")
    fm.write_cache_fp8(k, v, *(x[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")), table, none)
    check(run(x), x)
    assert fm.device_status() == 0


@pytest.mark.parametrize("t,h,g,d", [(1, 4, 1, 128), (6, 8, 2, 128), (3, 16, 2, 64), (5, 6, 1, 128)])
def test_queries_near_the_largest(t, h, g, d):
    """Scores of up to 2^123, which fp32 holds, as products of keys without their powers of two are not: the token with the largest has all the weight."""
    x = inputs(2, t, h, g, d, [300, 70], 16, torch.bfloat16, spread=0.0)
    x["q"], x["k"] = x["q"] * 2.0 ** 117, x["k"] * 2.0 ** -4
    out = run(x)
    assert out.isfinite().all()
    check(out, x)
