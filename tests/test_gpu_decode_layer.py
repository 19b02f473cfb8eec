"""The operators together: a decoder layer, token by token, against the same layer in FP32."""

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(device):
    spec = importlib.util.spec_from_file_location("decode_layer", Path(__file__).resolve().parents[1] / "examples" / "decode_layer.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("batch", [1, 4, 6])
def test_decode_layer(example, batch, bits):
    """BF16 (2^-8 for a rounding) between some ten steps, and 8-bit keys and values (at most half of 1 / 127
    of a row's largest); a token whose router hesitates between two experts may take the other one."""
    shape = example.Shape(hidden=512, heads=8, kv_heads=2, head_dim=64, experts=8, top_k=2, inter=256, max_tokens=64)
    assert example.compare(shape, batch, 40, bits) < 10 * 2.0 ** -8


def test_replayed_step(example):
    shape = example.Shape(hidden=512, heads=8, kv_heads=2, head_dim=64, experts=8, top_k=2, inter=256, max_tokens=64)
    assert example.time_step(shape, 2, 16, 8) > 0
