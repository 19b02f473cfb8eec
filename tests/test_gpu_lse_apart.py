"""`paged_attention` writes a head's sum while other heads' queries are read and other results written: an `lse` that lies over
either is refused, plain or shaped, by the short way and by the wrapper."""

import pytest
import torch

import chord_b200
from chord_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("shape", [{}, {"cap": 5.0}, {"slopes": True, "window": 9}])
def test_lse_over_what_is_read_or_written(device, monkeypatch, shape, short):
    if not short:
        monkeypatch.setattr(_lib, "direct", lambda: None)
    options = dict(shape)
    if "slopes" in options:
        options["slopes"] = torch.ones(6, device=device)
    cache = chord_b200.kv_cache(4, 16, 2, 64, device=device)
    table = torch.arange(4, dtype=torch.int32, device=device).view(4, 1)
    lengths = torch.tensor([3, 0, 16, 9], dtype=torch.int32, device=device)
    memory = torch.zeros(4096, dtype=torch.float32, device=device)
    q = memory[:768].view(torch.bfloat16).reshape(4, 6, 64)
    out = memory[1024:1792].view(torch.bfloat16).reshape(4, 6, 64)
    call = lambda **more: chord_b200.paged_attention(q, cache, table, lengths, **options, **more)  # noqa: E731
    for at in (0, 744, 767):
        with pytest.raises(ValueError, match="lse must not overlap q"):
            call(lse=memory[at:at + 24].view(4, 6))
        with pytest.raises(ValueError, match="lse must not overlap outputs"):
            call(lse=memory[1024 + at:1048 + at].view(4, 6), outputs=out)
    with pytest.raises(ValueError, match="lse must not overlap q"):
        call(lse=memory[760:784].view(4, 6), outputs=out)
    strided = memory[:1536].view(torch.bfloat16).reshape(4, 12, 64)[:, 3:9]  # (between its rows too: they are spanned)
    with pytest.raises(ValueError, match="lse must not overlap q"):
        chord_b200.paged_attention(strided, cache, table, lengths, lse=memory[320:344].view(4, 6), **options)
    lse = memory[768:792].view(4, 6)
    call(lse=lse)
    assert call(lse=memory[1792:1816].view(4, 6), outputs=out) is out
    assert torch.equal(lse, memory[1792:1816].view(4, 6))
    chord_b200.check_status(device)
