"""verify_drafts: an id that the draft gives as much as the target has nothing left once a sister of it was not accepted - exactly nothing, whatever r was divided by."""
import pytest
import torch

import fp6_marlin_b200 as fm
from test_gpu_verify_drafts import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("children,vocab", [(2, 1000), (5, 1000), (63, 4099)])
def test_as_much_in_the_draft_as_in_the_target(children, vocab, dtype):
    """The first child has no probability; the others have as much in both, and their drawn number is 0, with which anything that is left of theirs would be accepted."""
    b, t = 40, children + 1
    x = inputs(b, t, vocab, dtype, sharp=1.0)
    x["tree"] = fm.tree_masks(torch.tensor([-1] + [0] * children)).cuda()
    x["drafted"] = torch.stack([torch.randperm(vocab, generator=torch.Generator().manual_seed(s))[:t] for s in range(b)]).cuda()
    x["target"][:, 0].scatter_(1, x["drafted"][:, 1:2], 0.0)
    others = x["drafted"][:, 2:]
    x["target"][:, 0].scatter_(1, others, x["draft"][:, 0].gather(1, others))
    x["uniforms"][:, 1], x["uniforms"][:, 2:] = 0.5, 0.0
    got = check(x)
    assert (got[1] == 1).all()
