"""`cache_evict` takes scratch for the tokens that there can be, whatever the budget."""

import ctypes

import pytest
import torch

import chord_b200
from chord_b200 import _lib


@pytest.fixture(params=["native", "ctypes"])
def lib(request, native_lib):
    return _lib.native() if request.param == "native" else native_lib


def test_what_the_entry_asks_for(lib):
    at = 1 << 40  # (an aligned address that nothing is read from)
    cache = _lib.KVCacheDescriptor(k=at, v=at, k_scale=None, v_scale=None, num_pages=4, page_size=16, heads=2, head_dim=64, stride_page=2048,
                                   stride_head=1024, stride_token=64, scale_stride_page=0, scale_stride_head=0, scale_stride_token=0)

    def call(keep, width, size):
        arguments = [ctypes.addressof(cache), at, 4, 4, None, 0, 0, at, at, 2 * width, width, width, at, at, max(keep, width), at, size, None, 2, keep, 0, 0, None]
        return getattr(lib, "chord_b200_cache_evict")(*arguments), _lib.last_error()

    for keep, width in ((16, 64), (1 << 20, 64), ((1 << 28) - 1, 1), (64, 64)):
        needed = 2 * 2 * min(keep, width) * 4
        assert lib.chord_b200_cache_evict_workspace_bytes(2, 2, min(keep, width)) == needed
        code, message = call(keep, width, needed - 1)
        assert code == 1 and f"this launch needs {needed}" in message


@pytest.mark.gpu
@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("apart", [True, False])
def test_memory(device, monkeypatch, apart, short):
    if not short:
        monkeypatch.setattr(_lib, "direct", lambda: None)
    cache = chord_b200.kv_cache(12, 16, 8, 64, device=device)
    for x in (cache.k, cache.v):
        x.normal_()
    before = cache.k.clone()
    table, new = (torch.arange(6, dtype=torch.int32, device=device).add(i).reshape(2, 3) for i in (0, 6))
    lengths = torch.tensor([48, 5], dtype=torch.int32, device=device)
    weights, keep = torch.rand((2, 8, 48), device=device), 1 << 20
    held = keep * 2 * 8 * 4
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(device)
    start = torch.cuda.memory_allocated(device)
    got, kept = chord_b200.cache_evict(cache, table, lengths, weights, keep, new_tables=new if apart else None)
    assert torch.cuda.max_memory_allocated(device) - start < held + (1 << 20)
    assert got.tolist() == [48, 5] and torch.equal(kept[0, :, :48], weights[0]) and torch.equal(kept[1, :, :5], weights[1, :, :5])
    assert int(kept.count_nonzero()) == int(weights[0].count_nonzero() + weights[1, :, :5].count_nonzero())
    assert torch.equal(cache.k[:6], before[:6])
    if apart:
        assert torch.equal(cache.k[6:9], before[:3]) and torch.equal(cache.k[9, :, :5], before[3, :, :5])
    chord_b200.check_status(device)
