"""The same call gives the same bits, again and again, whatever the order in which warps and products come: items of many
steps and of one, cut and whole, of either kind of tile.  (A wait on a product that was two behind let the last step's
values be read before they were there, in 1 to 6 of 100 calls, for heads of 192 and 256.)"""

import pytest
import torch

import chord_b200
from tests.prompt_cases import Prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 8), (96, 6, 2), (128, 16, 2), (192, 8, 2), (256, 4, 2)])
def test_same_bits(device, dim, heads, kv_heads, bits):
    case = Prompt(device, [(20000, 9), (0, 700), (333, 20), (0, 1)], heads, kv_heads, dim, 16, bits, seed=heads)
    first, lse = case.run()
    different = torch.zeros((), dtype=torch.int64, device=device)
    for _ in range(300):
        sums = torch.empty_like(lse)
        out = chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, lse=sums)
        different += (out != first).sum() + (sums != lse).sum()
    assert int(different) == 0
    chord_b200.check_status(device)
