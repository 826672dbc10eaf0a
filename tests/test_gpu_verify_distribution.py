"""What the rule of verify_drafts gives for two sisters, exactly: the first token behind the last committed one over all pairs of sisters and over grids of drawn numbers that every border of the rule falls between.

p = (1, 9, 6) / 16, q = (8, 4, 4) / 16.  The first sister 0 is accepted for u < 1/8, 1 and 2 always; of r = (0, 5, 2) / 7 a second sister 1 or 2 is, 0 is not and leaves (0, 13, 1) / 14.  So eighths decide about
the first sister and fourteenths about the next token.
"""
from fractions import Fraction

import pytest
import torch

import fp6_marlin_b200 as fm
from test_gpu_verify_drafts import run

pytestmark = pytest.mark.gpu

P, Q = [Fraction(n, 16) for n in (1, 9, 6)], [Fraction(n, 16) for n in (8, 4, 4)]


def _shares(weight):
    """The probability of each first token, sisters a and b drawn with probability weight(a, b)."""
    grid = torch.cartesian_prod(torch.arange(3), torch.arange(3), torch.arange(8), torch.arange(14))
    n = len(grid)
    row = lambda values: torch.tensor([float(v) for v in values], device="cuda").expand(n, 3, 3).contiguous()          # noqa: E731
    uniforms = torch.stack([(grid[:, 3] + 0.5) / 14, (grid[:, 2] + 0.5) / 8, torch.full((n,), 0.5)], 1).cuda()
    drafted = torch.cat([torch.zeros((n, 1), dtype=torch.long), grid[:, :2]], 1).cuda()
    accepted, counts, next_tokens = run({"target": row(P), "draft": row(Q), "drafted": drafted, "uniforms": uniforms, "tree": fm.tree_masks(torch.tensor([-1, 0, 0])).cuda()})
    first = torch.where(counts > 1, drafted.gather(1, accepted[:, 1:2].clamp(min=0).long())[:, 0], next_tokens).tolist()
    shares = [Fraction(0)] * 3
    for (a, b, _, _), token in zip(grid.tolist(), first):
        shares[token] += weight(a, b) / (8 * 14)
    return shares


def test_sisters_that_were_drawn_independently_give_the_target():
    assert _shares(lambda a, b: Q[a] * Q[b]) == P


def test_sisters_that_were_drawn_without_repetition_do_not():
    """By how much is the rule's, too: the first sister as before, the second one never 0 after 0."""
    got = _shares(lambda a, b: Q[a] * Q[b] / (1 - Q[a]) if a != b else Fraction(0))
    # 0 first (1/2), accepted in an eighth of it; else 1 or 2 follow, half and half, and are accepted; 1 or 2 first (1/4 each): accepted
    assert got == [Fraction(1, 16), Fraction(1, 2) * Fraction(7, 8) / 2 + Fraction(1, 4), Fraction(1, 2) * Fraction(7, 8) / 2 + Fraction(1, 4)] and got != P
