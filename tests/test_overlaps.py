"""Results that would lie where a call still reads are refused."""

from pathlib import Path

import pytest
import torch

import chord_b200
from chord_b200 import _checks
from tests.cases import make_weights


def test_apart():
    room = torch.zeros(400)
    a = room[:100].view(10, 10)
    _checks.apart("a", a, "b", room[100:200])
    _checks.apart("a", a, "b", room[100:100])
    _checks.apart("a", a, "a", a, in_place=True)
    _checks.apart("a", a, "b", room.view(20, 20)[5:, :10])   # begins where a ends
    for other in (a, room[99:120], room[:1], room.view(20, 20)[:, 10:], a.t(), room[:50].view(5, 10)):
        with pytest.raises(ValueError, match="a must not overlap b"):
            _checks.apart("a", a, "b", other)
        if other is not a:
            with pytest.raises(ValueError, match="unless"):
                _checks.apart("a", a, "b", other, in_place=True)


@pytest.mark.gpu
def test_operators(device):
    codes, scale = make_weights(1, 128, 128, 5)
    w = chord_b200.pack_w4a16(codes.to(device), scale.to(device))
    room = torch.zeros((64, 128), dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="outputs must not overlap x"):
        chord_b200.gemv(room[:4], w, outputs=room[:4])
    with pytest.raises(ValueError, match="outputs must not overlap x"):
        chord_b200.gemv(room[:4], w, outputs=room[3:7])
    chord_b200.gemv(room[:4], w, outputs=room[4:8])
    cache = chord_b200.kv_cache(2, 16, 2, 64, device=device)
    rows = room.view(-1, 4, 64)
    table, ints = torch.zeros((2, 2), dtype=torch.int32, device=device), torch.ones(2, dtype=torch.int32, device=device)
    for out in (rows[:2], rows[1:3]):
        with pytest.raises(ValueError, match="outputs must not overlap q"):
            chord_b200.paged_attention(rows[:2], cache, table, ints, outputs=out)
    chord_b200.paged_attention(rows[:2], cache, table, ints, outputs=rows[2:4])
    weight, angles = torch.ones(64, dtype=torch.bfloat16, device=device), torch.zeros((8, 64), device=device)
    norm = (weight, weight, angles, ints)
    q, k = rows[:2], rows[2:4]
    for outs, message in ((dict(q_out=k), "q_out must not overlap k"), (dict(k_out=q), "k_out must not overlap q"),
                          (dict(q_out=rows[1:3]), "q_out must not overlap q"), (dict(q_out=rows[4:6], k_out=rows[5:7]), "q_out must not overlap k_out")):
        with pytest.raises(ValueError, match=message):
            chord_b200.qk_norm_rope(q, k, *norm, **outs)
    chord_b200.qk_norm_rope(q, k, *norm, q_out=q, k_out=k)
    kv = rows[4:6, :2]
    with pytest.raises(ValueError, match="q_out must not overlap v"):
        chord_b200.qk_norm_rope_write(q, rows[6:8, :2], kv, *norm, cache, ints, q_out=rows[4:6])
    chord_b200.qk_norm_rope_write(q, rows[6:8, :2], kv, *norm, cache, torch.tensor([0, 1], dtype=torch.int32, device=device), q_out=q)
    out = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="k_out must not overlap v_out"):
        chord_b200.cache_read(cache, table[:1], torch.tensor([0, 2], dtype=torch.int32, device=device), 2, k_out=out, v_out=out)
    chord_b200.check_status(device)


def test_what_is_said_of_slots():
    """Rows are written by several warps in no order, so nothing is promised of a slot that two tokens name."""
    header = (Path(__file__).resolve().parents[1] / "include" / "chord_b200.h").read_text()
    assert "leave either's row" not in header and "slots of a call are\n * distinct" in header
    for operator in (chord_b200.cache_write, chord_b200.qk_norm_rope_write):
        assert "distinct" in operator.__doc__
