"""Norms of heads over the sizes that are promised."""

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.test_gpu_heads import check, heads_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power,eps", [(-57, 0.0), (-57, 1e-6), (-20, 1e-12), (40, 1e-6), (57, 1e-6)])
@pytest.mark.parametrize("tokens", [5, 900])
def test_sizes(device, tokens, power, eps):
    q, k, _, qw, kw, table, positions = heads_case(device, tokens, 8, 2, 128, 64, seed=power + 100)
    q, k = ((x.double() * 2.0 ** power).to(torch.bfloat16) for x in (q, k))
    got = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions, eps=eps)
    for x, w, out in ((q, qw, got[0]), (k, kw, got[1])):
        check(out, A.norm_rope(x, w, table, positions, eps, False), x, w, table, positions, eps, False)
