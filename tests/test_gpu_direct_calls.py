"""The short ways through the wrappers give what the wrappers give, and leave to them what is not plain."""

import pytest
import torch

import chord_b200
from chord_b200 import _lib
from tests import attention_cases as A
from tests.cases import make_weights

pytestmark = pytest.mark.gpu


@pytest.fixture
def both(device, monkeypatch):
    """Runs a call through the module and without it; the results of both."""
    if _lib.direct() is None:
        pytest.skip("the module was not built")
    chord_b200.indexed_gemm.status_word(device)
    chord_b200.indexed_gemm.default_locks(device)

    def run(call, module_call=None):
        a = call()
        with monkeypatch.context() as m:
            m.setattr(_lib, "direct", lambda: None)
            b = call()
        for x, y in zip(*((r if isinstance(r, tuple) else (r,)) for r in (a, b))):
            assert x.shape == y.shape and x.stride() == y.stride() and torch.equal(x, y)
        return a

    return run


def test_results_agree(device, both):
    g = torch.Generator(device=device).manual_seed(1)
    codes, scale = make_weights(3, 256, 192, 5)
    weight = chord_b200.pack_w4a16(codes.to(device), scale.to(device))
    one = chord_b200.pack_w4a16(codes[:1].to(device), scale[:1].to(device))
    x = torch.randn((3, 400), generator=g, device=device).to(torch.bfloat16)[:, 200:392]
    ids = torch.tensor([[0, 4], [1, 2], [2, 0]], dtype=torch.int32, device=device)
    both(lambda: chord_b200.gemv(x, one))
    both(lambda: chord_b200.gemv(x, weight, expert_ids=ids, top_k=2))
    both(lambda: chord_b200.gemv(x, weight, expert_ids=ids, top_k=2, expert_base=1))

    qkv = torch.randn((5, 12, 64), generator=g, device=device).to(torch.bfloat16)
    q, k, v = qkv.split([8, 2, 2], dim=1)
    w = torch.rand(64, generator=g, device=device).to(torch.bfloat16)
    table, positions = A.angles(9, 32, device), torch.arange(5, dtype=torch.int32, device=device)
    slots = torch.arange(5, dtype=torch.int32, device=device)
    tables, offsets = torch.tensor([[0, 1, 0, 0]], dtype=torch.int32, device=device)[:, :3], torch.tensor([0, 5], dtype=torch.int32, device=device)
    for bits in (torch.bfloat16, torch.uint8):
        cache = chord_b200.kv_cache(2, 4, 2, 64, dtype=bits, device=device)
        for interleaved in (False, True):
            both(lambda: chord_b200.qk_norm_rope(q, k, w, w, table, positions, eps=1e-3, interleaved=interleaved))
            both(lambda: chord_b200.qk_norm_rope_write(q, k, v, w, w, table, positions, cache, slots, interleaved=interleaved))
        chord_b200.cache_write(k, v, cache, slots)
        both(lambda: chord_b200.cache_read(cache, tables, offsets, 6))
        lengths = torch.tensor([5], dtype=torch.int32, device=device)
        lse = torch.empty((1, 8), device=device)
        for options in ({}, {"window": 3}, {"scale": 0.25}, {"lse": lse}):
            both(lambda: chord_b200.paged_attention(q[4:], cache, tables, lengths, **options))


def test_what_is_left_to_the_wrapper(device, both):
    """Nothing unusual is taken: the module answers None, and the wrapper raises or copes."""
    module = _lib.direct()
    codes, scale = make_weights(1, 128, 64, 5)
    w = chord_b200.pack_w4a16(codes.to(device), scale.to(device))
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device=device)
    args = [x, w.packed, w.scale, 128, 64, 1, None, 1, 0]
    assert module.gemv(*args) is not None
    for at, value in ((0, x.float()), (0, x.cpu()), (0, x[:, :32]), (0, x[:0]), (0, torch.zeros((17, 64), dtype=torch.bfloat16, device=device)),
                      (1, w.packed.long()), (3, 256), (3, 128.0), (4, 128), (5, 2), (6, x), (6, torch.zeros(3, dtype=torch.int32, device=device)),
                      (7, 2), (7, True), (8, 1), (8, 1 << 80), (0, None), (1, "words")):
        wrong = list(args)
        wrong[at] = value
        assert module.gemv(*wrong) is None, (at, value)
    assert module.gemv(*args[:-1]) is None
    cache = chord_b200.kv_cache(2, 4, 2, 64, device=device)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=device)
    table, length = torch.zeros((1, 2), dtype=torch.int32, device=device), torch.ones(1, dtype=torch.int32, device=device)
    args = [q, cache.address, cache.index, table, length, None, 0, 0.125]
    assert module.paged_attention(*args) is not None
    for at, value in ((0, q[..., :32]), (0, q[:, :3]), (0, q[:, :0]), (2, 63), (3, table.long()), (3, table[:0]), (4, length[:0]), (5, length), (6, -1),
                      (6, 1 << 31), (7, float("nan")), (7, 1)):
        wrong = list(args)
        wrong[at] = value
        assert module.paged_attention(*wrong) is None, (at, value)
    odd = chord_b200.kv_cache(2, 4, 2, 80, device=device)
    assert module.paged_attention(torch.zeros((1, 4, 80), dtype=torch.bfloat16, device=device), odd.address, odd.index, table, length, None, 0, 1.0) is None


def test_another_stream_goes_through_the_wrapper_first(device):
    """A stream that has no lock buffer yet gets one, and later calls on it take the short way."""
    cache = chord_b200.kv_cache(2, 4, 2, 64, device=device)
    A.fill(cache, torch.Generator(device=device).manual_seed(0))
    q = torch.randn((1, 4, 64), device=device).to(torch.bfloat16)
    table, length = torch.tensor([[0, 1]], dtype=torch.int32, device=device), torch.tensor([7], dtype=torch.int32, device=device)
    want = chord_b200.paged_attention(q, cache, table, length)
    torch.cuda.synchronize(device)
    for _ in range(20):  # (more streams than the module remembers)
        stream = torch.cuda.Stream(device)
        with torch.cuda.stream(stream):
            for _ in range(2):
                got = chord_b200.paged_attention(q, cache, table, length)
        stream.synchronize()
        assert torch.equal(got, want)
