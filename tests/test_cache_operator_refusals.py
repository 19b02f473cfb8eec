"""What the operators over prompts, shared prefixes and evictions refuse without a GPU."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

import chord_b200
from chord_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]
AT = 1 << 40  # an aligned address that nothing is read from


def test_operators_want_a_cache():
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: chord_b200.prompt_attention(q, None, i, i, i),
                 lambda: chord_b200.shared_prefix_attention(q, "cache", i, i, i, i, i),
                 lambda: chord_b200.attention_weights(q, q, i, i, q),
                 lambda: chord_b200.cache_evict(None, i, i, q, 4),
                 lambda: chord_b200.paged_attention(q, None, i, i, cap=30.0)):
        with pytest.raises(TypeError, match="KVCache"):
            call()


def test_scores_are_the_header_s():
    text = (ROOT / "include" / "chord_b200.h").read_text()
    body = re.search(r"typedef struct chord_b200_scores \{(.*?)\}", text, re.S).group(1)
    names = [n.strip(" *") for line in body.split(";")
             for n in re.sub(r"^\s*(const float\*|double|int64_t)", "", line.strip()).split(",") if n.strip()]
    assert [name for name, _ in _lib.ScoresDescriptor._fields_] == names
    assert ctypes.sizeof(_lib.ScoresDescriptor) == 8 * len(names)


def cache(**changes):
    fields = dict(k=AT, v=AT, k_scale=None, v_scale=None, num_pages=4, page_size=16, heads=2, head_dim=64, stride_page=2048,
                  stride_head=1024, stride_token=64, scale_stride_page=0, scale_stride_head=0, scale_stride_token=0)
    return _lib.KVCacheDescriptor(**{**fields, **changes})


def refused(lib, name, good, wrong):
    for place, value, message in wrong:
        arguments = list(good)
        arguments[place] = value
        assert getattr(lib, name)(*arguments) == 1, (name, place, value)
        assert message in _lib.last_error(), (name, place, value, _lib.last_error())


SCORES = [  # what is wrong with them, whichever entry has them
    ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"cap": -1.0}, "cap"), ({"cap": float("nan")}, "cap"),
    ({"cap": 1e-31}, "cap"), ({"cap": 1e31}, "cap"), ({"cap": 1.0, "scale": 1e37}, "cap"), ({"window": -1}, "window"),
    ({"window": 1 << 31}, "window"),
]


def wrong_scores(place, kept):
    made = []
    for change, message in SCORES:
        kept.append(_lib.ScoresDescriptor(**{**dict(scale=0.125, cap=0.0, slopes=None, window=0), **change}))
        made.append((place, ctypes.addressof(kept[-1]), message))
    return made


@pytest.fixture(params=["native", "ctypes"])
def lib(request, native_lib):
    return _lib.native() if request.param == "native" else native_lib


def test_prompts(lib):
    kept = [cache(), cache(head_dim=80), cache(v=AT + 8), _lib.ScoresDescriptor(0.125, 0.0, None, 0)]
    good = [AT, 256, 64, ctypes.addressof(kept[0]), AT, 4, 4, AT, AT, None, None, AT, None, AT, 1 << 40, None, 2, 8, 4,
            ctypes.addressof(kept[3]), None]
    refused(lib, "chord_b200_prompt_attention", good,
            [(0, None, "null"), (4, None, "null"), (7, None, "null"), (8, None, "null"), (11, None, "null"), (13, None, "null"), (19, None, "null"),
             (1, 12, "16-byte"), (2, -64, "16-byte"), (0, AT + 2, "16-byte"), (11, AT + 8, "16-byte"), (13, AT + 4, "16-byte"),
             (3, ctypes.addressof(kept[1]), "head_dim"), (3, ctypes.addressof(kept[2]), "aligned"), (6, 0, "page"), (5, -1, "page"),
             (18, 3, "multiple"), (18, 0, "multiple"), (17, 1 << 31, "sizes"), (17, 1 << 30, "too many")] + wrong_scores(19, kept))
    size = lib.chord_b200_prompt_attention_workspace_bytes
    assert size(-1, 8, 4, 2, 64) == -1 and size(2, 8, 3, 2, 64) == -1 and size(2, 8, 4, 2, 80) == -1


def test_shared_prefixes(lib):
    kept = [cache(), cache(head_dim=80), _lib.ScoresDescriptor(0.125, 0.0, None, 0)]
    good = [AT, 256, 64, ctypes.addressof(kept[0]), AT, 4, 4, AT, AT, 2, AT, 4, 4, AT, AT, None, AT, 1024, AT, 1 << 40, None, 8, 4,
            ctypes.addressof(kept[2]), None]
    refused(lib, "chord_b200_shared_prefix_attention", good,
            [(place, None, "null") for place in (0, 4, 7, 8, 10, 13, 14, 16, 23)] +
            [(18, None, "workspace"), (1, 12, "16-byte"), (3, ctypes.addressof(kept[1]), "head_dim"), (6, 0, "page"), (12, 0, "page"), (22, 3, "multiple")] +
            wrong_scores(23, kept))


def test_weights(lib):
    kept = [cache(), cache(head_dim=80), _lib.ScoresDescriptor(0.125, 0.0, None, 0)]
    good = [AT, 256, 64, ctypes.addressof(kept[0]), AT, 4, 4, AT, AT, AT, 128, 64, 64, 0, None, 2, 4, ctypes.addressof(kept[2]), None]
    refused(lib, "chord_b200_attention_weights", good,
            [(place, None, "null") for place in (0, 4, 7, 8, 9, 17)] +
            [(1, 12, "16-byte"), (3, ctypes.addressof(kept[1]), "head_dim"), (6, 0, "page"), (10, -1, "sizes"), (12, 1 << 31, "sizes"),
             (15, -1, "batch"), (15, 65536, "batch"), (16, 3, "multiple")] + wrong_scores(17, kept))


def test_evictions(lib):
    kept = [cache(), cache(num_pages=0)]
    good = [ctypes.addressof(kept[0]), AT, 4, 4, None, 0, 0, AT, AT, 128, 64, 64, AT, AT, 64, AT, 1 << 40, None, 2, 16, 2, 2, None]
    refused(lib, "chord_b200_cache_evict", good,
            [(place, None, "null") for place in (1, 7, 8, 12, 13, 15)] +
            [(0, ctypes.addressof(kept[1]), "tokens"), (3, 0, "page"), (4, AT, "page"), (11, 0, "sizes"), (14, 15, "sizes"), (15, AT + 2, "workspace"),
             (16, 2 * 2 * 16 * 4 - 1, "workspace"), (18, -1, "batch"), (18, 65536, "batch"), (19, 0, "keep"), (19, 1 << 28, "keep"),
             (20, -1, "first"), (20, 15, "first"), (21, -1, "first"), (21, 15, "first")])
    size = lib.chord_b200_cache_evict_workspace_bytes
    assert size(2, 2, 16) == 256 and size(-1, 2, 16) == -1 and size(1 << 16, 2, 16) == -1 and size(2, 2, 1 << 28) == -1
