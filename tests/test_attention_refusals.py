"""What the attention-side operators refuse without a GPU: types first, then places, shapes and layouts."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

import chord_b200
from chord_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_cache_tensors():
    k = torch.zeros((2, 1, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="k must be torch.bfloat16"):
        chord_b200.KVCache(k.float(), k.float())
    with pytest.raises(TypeError, match="k must be torch.uint8"):
        chord_b200.KVCache(k, k, torch.zeros((2, 1, 4)), torch.zeros((2, 1, 4)))
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        chord_b200.KVCache(None, k)
    with pytest.raises(ValueError, match="CUDA"):
        chord_b200.KVCache(k, k)
    with pytest.raises(ValueError, match="4D"):
        chord_b200.KVCache(k[0], k[0])


def test_cache_sizes():
    for wrong in ((0, 16, 2, 64), (4, -1, 2, 64), (4, 16, True, 64), (4, 16, 2, 64.0)):
        with pytest.raises(ValueError, match="must be"):
            chord_b200.kv_cache(*wrong, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        chord_b200.kv_cache(4, 16, 2, 64, dtype=torch.float16, device="cpu")


def test_operators_want_tensors_on_the_gpu():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="x must be"):
        chord_b200.gemv(x.float(), None)
    with pytest.raises(ValueError, match="CUDA"):
        chord_b200.gemv(x, None)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        chord_b200.qk_norm_rope(q, q, x[0], x[0], x.float(), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="q must be"):
        chord_b200.qk_norm_rope(x, q, x[0], x[0], x.float(), torch.zeros(2, dtype=torch.int32))
    for call in (lambda: chord_b200.paged_attention(q, None, None, None), lambda: chord_b200.cache_write(q, q, None, None),
                 lambda: chord_b200.cache_read(None, None, None, 1),
                 lambda: chord_b200.qk_norm_rope_write(q, q, q, x, x, x, x, "cache", x)):
        with pytest.raises(TypeError, match="KVCache"):
            call()


def test_descriptor_is_the_header_s():
    text = (ROOT / "include" / "chord_b200.h").read_text()
    body = re.search(r"typedef struct chord_b200_kv_cache \{(.*?)\}", text, re.S).group(1)
    names = [n.strip(" *") for line in body.split(";") for n in re.sub(r"^\s*(void\*|float\*|int64_t)", "", line.strip()).split(",") if n.strip()]
    assert [name for name, _ in _lib.KVCacheDescriptor._fields_] == names
    assert ctypes.sizeof(_lib.KVCacheDescriptor) == 8 * len(names)


def test_c_entries_refuse_before_they_look_for_a_gpu(native_lib):
    native = _lib.native()
    at = 1 << 40
    gemv = [at, 64, at, at, None, at, 1, 128, 64, 1, 1, 0, None]
    for place, value, message in ((0, None, "null"), (1, 63, "apart"), (2, at + 4, "aligned"), (6, 17, "rows"), (6, -1, "rows"), (7, 100, "n must"),
                                  (8, 96, "k must"), (9, 0, "num_experts"), (10, 0, "top_k"), (11, -1, "expert_base")):
        wrong = list(gemv)
        wrong[place] = value
        for lib in (native, native_lib):
            assert lib.chord_b200_gemv(*wrong) == 1
            assert message in _lib.last_error()
    fields = dict(k=at, v=at, k_scale=None, v_scale=None, num_pages=4, page_size=16, heads=2, head_dim=64, stride_page=2048,
                  stride_head=1024, stride_token=64, scale_stride_page=0, scale_stride_head=0, scale_stride_token=0)
    for change, message in (({"k": None}, "null"), ({"v_scale": at}, "scales"), ({"num_pages": 0}, "tokens"), ({"num_pages": 1 << 28}, "tokens"),
                            ({"heads": 0}, "heads"), ({"head_dim": 72}, "head_dim"), ({"head_dim": 272}, "head_dim"), ({"stride_token": 65}, "multiples"),
                            ({"stride_page": -2048}, "multiples"), ({"v": at + 8}, "aligned"), ({"stride_page": 1 << 36}, "2^36")):
        cache = _lib.KVCacheDescriptor(**{**fields, **change})
        address = ctypes.addressof(cache)
        attend = (at, 256, 64, address, at, 4, 4, at, at, None, at, 1024, at, 1 << 30, None, 1, 4, 0, 0.125, None)
        for lib in (native, native_lib):
            assert lib.chord_b200_paged_attention(*attend) == 1
            assert message in _lib.last_error(), (change, _lib.last_error())
            assert lib.chord_b200_cache_write(at, 128, 64, at, 128, 64, address, at, 1, None, None) == 1
            assert lib.chord_b200_cache_read(address, at, 4, 4, at, 1, at, at, 1, None, None) == 1
    cache = _lib.KVCacheDescriptor(**fields)
    good = [at, 256, 64, ctypes.addressof(cache), at, 4, 4, at, at, None, at, 1024, at, 1 << 30, None, 1, 4, 0, 0.125, None]
    for place, value, message in ((0, None, "null"), (1, 12, "16-byte"), (6, 0, "page"), (16, 3, "multiple"), (17, -1, "window"), (18, float("nan"), "scale"),
                                  (18, float("inf"), "scale")):
        wrong = list(good)
        wrong[place] = value
        for lib in (native, native_lib):
            assert lib.chord_b200_paged_attention(*wrong) == 1
            assert message in _lib.last_error(), (place, _lib.last_error())
    rotate = [at, 256, 64, at, 128, 64, at, at, at, 10, 64, 0, at, at, at, 1, 4, 2, 64, None, 1e-6, None]
    for place, value, message in ((0, None, "null"), (1, 4, "q must"), (4, 4, "k must"), (6, at + 2, "aligned"), (9, 0, "position"), (10, 24, "rotary"),
                                  (10, 80, "rotary"), (12, None, "null"), (14, None, "k_out"), (16, 0, "heads"), (18, 40, "head_dim"), (20, -1.0, "eps"),
                                  (20, float("nan"), "eps")):
        wrong = list(rotate)
        wrong[place] = value
        for lib in (native, native_lib):
            assert lib.chord_b200_qk_norm_rope(*wrong) == 1
            assert message in _lib.last_error(), (place, _lib.last_error())


@pytest.mark.skipif(_lib._call is None, reason="the call module was not built")
def test_doubles_are_doubles(native_lib):
    with pytest.raises(TypeError):
        _lib.native().chord_b200_qk_norm_rope(*range(20), "1e-6", None)
    with pytest.raises(TypeError, match="takes 22 arguments"):
        _lib.native().chord_b200_qk_norm_rope(*range(21))
