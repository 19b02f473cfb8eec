"""Where the results of `prompt_attention` and `shared_prefix_attention` go: into any rows on 16-byte boundaries, and nowhere else."""

import pytest
import torch

import chord_b200
from tests.prompt_cases import Prompt
from tests.test_gpu_shared_prefix import Shared

pytestmark = pytest.mark.gpu


def behind(x, by):
    """A tensor like x, `by` elements behind a 256-byte boundary, between elements that are to be left."""
    room = torch.full((x.numel() + by + 64,), 7.0, dtype=torch.bfloat16, device=x.device)
    return room, room[by:by + x.numel()].view(x.shape)


def left(room, out, by):
    return bool((room[:by] == 7).all()) and bool((room[by + out.numel():] == 7).all())


@pytest.mark.parametrize("by", [8, 16, 24])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_outputs_on_16_bytes(device, dim, bits, by):
    """8 and 24 elements: on 16 bytes, not on 32.  Items that are whole, and some that are cut and joined."""
    for sequences in ([(0, 150), (40, 33), (0, 1)], [(9000, 9), (0, 40)]):
        case = Prompt(device, sequences, 6, 2, dim, 16, bits, seed=dim)
        want, _ = case.run()
        room, out = behind(want, by)
        assert out.data_ptr() % 32 == 2 * by % 32
        result = chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, outputs=out)
        chord_b200.check_status(device)
        assert result is out and torch.equal(out, want) and left(room, out, by)
    case = Shared(device, [(100, [3, 0, 40]), (0, [5])], 8, 2, dim, 16, bits, seed=dim)
    want, _ = case.run()
    room, out = behind(want, by)
    chord_b200.shared_prefix_attention(case.q, case.cache, case.prefix_table, case.prefix_lengths, case.offsets, case.table,
                                       case.lengths, outputs=out)
    chord_b200.check_status(device)
    assert torch.equal(out, want) and left(room, out, by)
