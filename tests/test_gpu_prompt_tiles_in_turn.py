"""Items of one row tile and of two in turn, long ones before short ones, over codes whose pages no box divides: the warps of the
second tile go past whole items without waiting for anything of theirs, and take the scales of the next one's steps when
these are there, not before.  (They went by a parity that the item before could have left.)"""

import pytest
import torch

import chord_b200
from tests.prompt_cases import Prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("heads", [24, 32])
@pytest.mark.parametrize("dim,page", [(64, 25), (96, 25), (96, 26), (128, 25)])
def test_scales_of_the_second_tile(device, dim, page, heads, cap):
    """24 heads: queries by the warps that bring the scales as well; 32: by TMA.  30 new tokens of three or four heads are one tile of 9
    steps.  Some 22 steps for a CTA, of 17 or 18 in a pair of sequences: every run crosses items of either kind.  (Pages of 25 are not divided by boxes of 2; of heads of 128 they are
    loaded in boxes of one.)"""
    case = Prompt(device, [(1100, 30), (0, 300)] * 24, heads, 8, dim, page, 8, seed=dim + heads)
    out, lse = case.check(cap=cap)
    different = torch.zeros((), dtype=torch.int64, device=device)
    for _ in range(50):
        again = torch.empty_like(lse)
        different += (chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, cap=cap, lse=again) != out).sum()
        different += (again != lse).sum()
    assert int(different) == 0
    chord_b200.check_status(device)
