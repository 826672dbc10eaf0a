"""verify_drafts by clusters of sixteen CTAs down to one: how many there are follows from the batch, and from what a device has room for, and changes no result."""
import pytest
import torch

from test_gpu_verify_drafts import check, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_sequence_in_batches_of_any_size(dtype, with_draft):
    x = inputs(2, 5, 70001, dtype, with_draft)
    want = check(x)
    for b in (8, 18, 19, 56, 64, 100, 148, 220, 300, 444, 500):    # 16, 16, 8, 7, 6, 4, 3, 2, 1, 1, 1 CTAs a sequence on 148 multiprocessors
        y = {n: None if v is None else v.repeat(-(-b // 2), *([1] * (v.dim() - 1)))[:b] for n, v in x.items()}
        for got, expect in zip(run(y), want):
            assert torch.equal(got, expect.repeat(-(-b // 2), *([1] * (expect.dim() - 1)))[:b])
