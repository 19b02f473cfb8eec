"""`gemv` over inputs at the ends of their type: results that are finite come out finite."""

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.test_gpu_gemv import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-110, -60, 60, 120, 127])
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 16])
def test_inputs_of_every_size(device, rows, power):
    """Codes of one sign and inputs just below 2^(power + 1), so that nothing cancels; scales bring the results near one."""
    n, k = 128, 192
    g = torch.Generator().manual_seed(rows + power + 200)
    codes = torch.randint(13, 16, (1, n, k), generator=g, dtype=torch.int32)
    codes[:, ::2] = 15 - codes[:, ::2]
    scale = ((torch.rand((1, n, k // 32), generator=g) + 0.5).double() * 2.0 ** max(-power, -110)).to(torch.bfloat16)
    x = ((torch.rand((rows, k), generator=g) * 0.9 + 1).double() * 2.0 ** power).to(torch.bfloat16)
    codes, scale, x = codes.to(device), scale.to(device), x.to(device)
    assert bool(torch.isfinite(x).all())
    got = chord_b200.gemv(x, chord_b200.pack_w4a16(codes, scale))
    want, size = A.gemv(x, codes, scale)
    assert bool(torch.isfinite(got).all())
    check(got, want, size, k)


def test_one_expert_s_row(device):
    n, k = 128, 256
    codes = torch.full((2, n, k), 15, dtype=torch.int32, device=device)
    scale = torch.full((2, n, k // 32), 2.0 ** -60, dtype=torch.bfloat16, device=device)
    weight = chord_b200.pack_w4a16(codes, scale)
    x = torch.full((1, k), 3.0e38, dtype=torch.bfloat16, device=device)
    got = chord_b200.gemv(x, weight, expert_ids=torch.tensor([1, 0], dtype=torch.int32, device=device), top_k=2)
    want, size = A.gemv(x, codes, scale, torch.tensor([1, 0]), 2)
    check(got, want, size, k)
