"""Scales at the edges of FP32 and beyond."""

import pytest
import torch

from tests.prompt_cases import Prompt
from tests.test_gpu_shared_prefix import Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 192])
@pytest.mark.parametrize("scale", [1e-40, 1e-46, 5e-324, -1e-46])
def test_scales_that_fp32_does_not_hold(device, scale, dim, bits):
    """So near zero, every token that a row sees has the same weight, and the others none."""
    Prompt(device, [(0, 140), (30, 20)], 4, 2, dim, 16, bits, seed=1).check(scale=scale)
    Shared(device, [(100, [20, 0])], 4, 2, dim, 16, bits, seed=1).check(scale=scale)
