"""The extension module that holds code of torch's headers is used with that torch only."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from chord_b200 import _lib, build

ROOT = Path(__file__).resolve().parents[1]
needs_module = pytest.mark.skipif(not build._torch_module_path().exists(), reason="the module was not built")


def test_version_is_torch_s():
    assert build._torch_version() == torch.__version__


@needs_module
def test_another_torch_makes_it_stale(native_lib, monkeypatch):
    assert build.is_fresh()
    monkeypatch.setattr(build, "_torch_version", lambda: torch.__version__ + "1")
    assert not build.is_fresh()
    monkeypatch.setattr(build, "_torch_version", lambda: torch.__version__[:-1])
    assert not build.is_fresh()


@needs_module
def test_another_torch_does_not_use_it(native_lib):
    code = ("import torch, warnings; torch.__version__ = '0.1'\n"
            "with warnings.catch_warnings(record=True) as said:\n"
            "    warnings.simplefilter('always')\n"
            "    from chord_b200 import _lib\n"
            "assert _lib.direct() is None and 'another torch' in str(said[0].message)")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    if _lib._torch_call is not None:
        assert _lib._torch_call.built_for == f"built for torch {torch.__version__}"
