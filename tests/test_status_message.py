"""What check_status says of a status word: all that its bits stand for."""

import pytest
import torch

from chord_b200 import indexed_gemm


@pytest.mark.parametrize("bits,names,index", [(1, ["producer wait"], False), (18, ["MMA-issuer wait", "stream-K lock wait"], False),
                                              (32, [], True), (34, ["MMA-issuer wait"], True), (63, ["epilogue wait", "producer wait"], True)])
def test_message(bits, names, index, monkeypatch):
    word = torch.tensor([bits], dtype=torch.int32)
    monkeypatch.setitem(indexed_gemm._STATUS, 63, word)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: None)
    with pytest.raises(RuntimeError) as raised:
        indexed_gemm.check_status("cuda:63")
    said = str(raised.value)
    assert all(name in said for name in names) and f"status {bits}" in said
    assert ("bounded wait" in said) == bool(names) and ("index outside a cache" in said) == index
    assert int(word) == 0
    indexed_gemm.check_status("cuda:63")
