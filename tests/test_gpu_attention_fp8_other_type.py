"""tree_attention_fp8 with more than 32 rows of a head of keys over a cache that was not written from the type of the queries: powers of two that fp16 does not hold are reported."""
import pytest
import torch

import fp6_marlin_b200 as fm
from test_gpu_tree_attention_fp8 import check, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,h,g,d", [(6, 8, 1, 128), (20, 8, 2, 64), (40, 32, 4, 128), (64, 64, 8, 128)])
@pytest.mark.parametrize("page", [16, 12])
def test_exponents_of_another_type(t, h, g, d, page):
    for name in ("k_scales", "v_scales"):
        for at in (0, 70, 899):
            x = inputs(2, t, h, g, d, [900, 70], page)
            where = (int(x["page_table"][0, at // page]), at % page, g - 1)
            for exponent, status in ((-24, 0), (15, 0), (-25, 4), (16, 4), (-127, 4), (127, 4)):
                x[name][where] = exponent + 127
                run(x)
                assert fm.device_status() == status, (name, at, exponent)
    x = inputs(2, t, h, g, d, [900, 70], page, fill=255)           # what is not read is not reported
    check(run(x), x)
    assert fm.device_status() == 0
