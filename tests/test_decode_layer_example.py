"""The decoder layer's example refuses what its tables have no room for, before anything runs on a GPU."""

import importlib.util
import sys
from pathlib import Path

import pytest
import torch


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decode_layer_host", Path(__file__).resolve().parents[1] / "examples" / "decode_layer.py")
    module = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = module
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("batch,steps", [(1, 61), (1, 0), (1, 512), (0, 8), (17, 8)])
def test_sizes(example, batch, steps, monkeypatch):
    shape = example.Shape(max_tokens=64)
    monkeypatch.setattr(example, "DecodeLayer", None)   # nothing is built
    for call in (example.compare, example.time_step):
        with pytest.raises(ValueError, match="must be from 1 to"):
            call(shape, batch, steps, 8)


def test_command_line(example, monkeypatch, capsys):
    monkeypatch.setattr(example, "DecodeLayer", None)
    monkeypatch.setattr(sys, "argv", ["decode_layer.py", "--steps", "600"])
    with pytest.raises(SystemExit) as stopped:
        example.main()
    assert stopped.value.code == 2 and "steps must be from 1 to 508" in capsys.readouterr().err


def test_slots_past_the_table(example):
    tables = torch.tensor([[5, 2, 7], [1, 0, 3]], dtype=torch.int32)
    positions = torch.tensor([47, 16], dtype=torch.int32)
    assert example.slots_for(tables, positions, 16).tolist() == [7 * 16 + 15, 0]
    for past in (48, 64, 2**31 - 1, -1):
        got = example.slots_for(tables, torch.tensor([past, 0], dtype=torch.int32), 16)
        assert got.dtype == torch.int32 and got.tolist() == [-1, 16]
