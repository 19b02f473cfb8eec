"""The package's modules are there as its attributes, whichever name was used first."""

import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("name", ["indexed_gemm", "grouped_gemm"])
def test_module_as_an_attribute(name):
    code = f"import chord_b200; assert chord_b200.{name}.__name__ == 'chord_b200.{name}'"
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_unknown_names():
    import chord_b200

    for name in ("no_such_operator", "csrc", "__wrapped__"):
        with pytest.raises(AttributeError):
            getattr(chord_b200, name)
