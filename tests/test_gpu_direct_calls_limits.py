"""Numbers that no call has are left to the wrapper, which refuses them."""

import pytest
import torch

import chord_b200
from chord_b200 import _lib
from tests.cases import make_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k", [65536, 1 << 31, 1 << 62, (1 << 63) - 1])
def test_more_routes_than_there_can_be(device, top_k):
    codes, scale = make_weights(2, 128, 64, 5)
    w = chord_b200.pack_w4a16(codes.to(device), scale.to(device))
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=device)
    ids = torch.zeros(0, dtype=torch.int32, device=device)   # (as many as 4 << 62 in 64 bits)
    chord_b200.gemv(x, w, expert_ids=torch.zeros(4, dtype=torch.int32, device=device))
    if _lib.direct() is not None:
        assert _lib.direct().gemv(x, w.packed, w.scale, 128, 64, 2, ids, top_k, 0) is None
    with pytest.raises(ValueError, match="expert_ids must hold"):
        chord_b200.gemv(x, w, expert_ids=ids, top_k=top_k)
