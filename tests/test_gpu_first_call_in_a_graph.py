"""`gemv` needs nothing that would have to be allocated in a capture: its first call on a device may be captured."""

import pytest
import torch

import chord_b200
from chord_b200 import _lib, indexed_gemm
from tests.cases import make_weights

pytestmark = pytest.mark.gpu


def test_first_call_in_a_graph(device, monkeypatch):
    codes, scale = make_weights(1, 256, 128, 5)
    weight = chord_b200.pack_w4a16(codes.to(device), scale.to(device))
    x = torch.randn((2, 128), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
    want = chord_b200.gemv(x, weight)
    torch.cuda.synchronize(device)
    monkeypatch.setattr(indexed_gemm, "_STATUS", {})
    monkeypatch.setattr(_lib, "direct", lambda: None)   # a device that the short way does not know
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chord_b200.gemv(x, weight)
    assert not indexed_gemm._STATUS
    graph.replay()
    assert torch.equal(out, want)
    chord_b200.gemv(x, weight)
    assert indexed_gemm._STATUS     # (from here on the short way is open)
