"""A row of `prompt_attention` depends, bit for bit, on what it sees alone: not on later tokens of its sequence that others
of the same tile see, nor on what lies in memory that no row sees.  (Finite ones; infinities and NaN change how weights are rounded.)"""

import pytest
import torch

import chord_b200
from tests.test_gpu_prompt_attention import Prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", [{}, {"cap": 20.0}, {"cap": 3.0, "lean": True}])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_later_tokens(device, dim, shape, bits):
    case = Prompt(device, [(70, 200), (0, 90)], 8, 2, dim, 16, bits, seed=23)
    options = {k: v for k, v in shape.items() if k != "lean"}
    if "lean" in shape:
        options["slopes"] = torch.linspace(0.01, 0.5, 8, device=device)
    clean = case.run(**options)
    page, place = (lambda t: int(case.table[0, t // 16])), (lambda t: t % 16)
    for late in (269, 200, 135):  # keys that raise the scores far above those before, from one token on
        at = page(late), slice(None), place(late)
        if bits == 8:
            case.cache.k_scale[at] *= 40.0
        else:
            case.cache.k[at] *= 40.0
        out, lse = case.run(**options)
        rows = list(range(late - 70)) + list(range(200, 290))
        assert torch.equal(out[rows], clean[0][rows]) and torch.equal(lse[rows], clean[1][rows])
        assert not torch.equal(lse[late - 70:200], clean[1][late - 70:200])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page", [16, 7])
def test_heads_that_are_one(device, page, bits):
    """A cache whose heads are views of one: strides of zero."""
    case = Prompt(device, [(20, 60), (0, 33)], 4, 2, 64, page, bits, seed=29)
    parts = [case.cache.k, case.cache.v] + ([case.cache.k_scale, case.cache.v_scale] if bits == 8 else [])
    for x in parts:
        x[:, 1] = x[:, 0]
    want = case.run()
    case.cache = chord_b200.KVCache(*(x[:, :1].expand(x.shape) for x in parts))
    got = case.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
