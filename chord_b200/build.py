"""Ahead-of-time build of ``libchord_b200.so`` (sm_100a only) with nvcc.

The reference compiles its kernels at run time through NVRTC
(chord_kernels/operator/jit/compiler.py:51-105); here every kernel is compiled
once, in-tree, and linked into one C-ABI shared library.  Run as
``python -m chord_b200.build``.
"""

from __future__ import annotations

import concurrent.futures
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
CSRC = PACKAGE_DIR / "csrc"
LIB_PATH = PACKAGE_DIR / "libchord_b200.so"
SOURCES = ("core.cu", "gemm.cu", "pack.cu", "fused.cu", "ep.cu", "gemv.cu", "heads.cu", "attention.cu")
ARCH_FLAGS = ("-gencode", "arch=compute_100a,code=sm_100a")


def _nvcc() -> str:
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")
    return nvcc


def _newest_source_mtime() -> float:
    files = [f for kind in ("cu", "cuh", "h", "c") for f in CSRC.glob("*." + kind)]
    files.append(PACKAGE_DIR.parent / "include" / "chord_b200.h")
    return max(f.stat().st_mtime for f in files if f.exists())


def is_fresh() -> bool:
    return (LIB_PATH.exists() and LIB_PATH.stat().st_mtime >= _newest_source_mtime() and _call_module_is_fresh()
            and _torch_module_is_fresh())


def _call_module_path() -> Path:
    return PACKAGE_DIR / ("_call" + sysconfig.get_config_var("EXT_SUFFIX"))


def _call_compiler() -> list[str] | None:
    """What compiles the `_call` module, or None where that cannot be done here."""
    headers = Path(sysconfig.get_paths()["include"])
    gcc = shutil.which(os.environ.get("CC", "gcc"))
    return [gcc, f"-I{headers}"] if gcc is not None and (headers / "Python.h").exists() else None


def _call_module_is_fresh() -> bool:
    """Up to date, or not to be had here (the library is then called through ctypes)."""
    path = _call_module_path()
    if path.exists():
        return path.stat().st_mtime >= (CSRC / "pycall.c").stat().st_mtime
    return _call_compiler() is None


def _compile(nvcc: str, src: str, obj_dir: Path, verbose: bool) -> Path:
    obj = obj_dir / (src + ".o")
    cmd = [
        nvcc, *ARCH_FLAGS, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
        "-Xptxas", "-v" if verbose else "-warn-spills",
        "-c", str(CSRC / src), "-o", str(obj),
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{proc.stdout}\n{proc.stderr}")
    if verbose:
        sys.stderr.write(proc.stderr)
    return obj


def _build_call_module() -> None:
    """The optional ``_call`` extension module (csrc/pycall.c); without Python's headers or a C
    compiler the library is called through ctypes instead, which is slower, hence the warning."""
    out = _call_module_path()
    compiler = _call_compiler()
    reason = "no C compiler or no Python headers"
    if compiler is not None:
        tmp = out.with_suffix(".tmp")
        cmd = [*compiler, "-O2", "-Wall", "-fPIC", "-shared", str(CSRC / "pycall.c"), "-o", str(tmp)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode == 0:
            os.replace(tmp, out)
            return
        reason = proc.stderr
    out.unlink(missing_ok=True)  # not one of another version
    warnings.warn(f"chord_b200._call was not built, calls go through ctypes (some 4 us each): {reason}")


def _torch_module_path() -> Path:
    return PACKAGE_DIR / ("_torch_call" + sysconfig.get_config_var("EXT_SUFFIX"))


def _torch_version() -> str | None:
    """``torch.__version__`` of the torch that would be imported, without importing it."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        return None
    found = re.search(r"^__version__ = ['\"](.+)['\"]$", (Path(spec.origin).parent / "version.py").read_text(), re.M)
    return found.group(1) if found else None


def _torch_compiler() -> list[str] | None:
    """What compiles the `_torch_call` module, without its source and output, or None where that
    cannot be done here."""
    spec = importlib.util.find_spec("torch")
    gxx = shutil.which(os.environ.get("CXX", "g++"))
    if spec is None or spec.origin is None or gxx is None:
        return None
    torch = Path(spec.origin).parent
    cuda = Path(_nvcc()).resolve().parents[1] / "include"
    headers = [Path(sysconfig.get_paths()["include"]), torch / "include", torch / "include/torch/csrc/api/include", cuda]
    if not all((headers[i] / name).exists() for i, name in ((0, "Python.h"), (1, "ATen/cuda/EmptyTensor.h"),
                                                            (3, "cuda_runtime_api.h"))):
        return None
    libraries = ["torch_python", "torch_cuda", "torch_cpu", "c10_cuda", "c10"]
    return [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", f'-DCHORD_TORCH_VERSION="{_torch_version()}"', *(f"-I{h}" for h in headers), f"-L{torch / 'lib'}",
            *(f"-l{name}" for name in libraries)]


def _torch_module_is_fresh() -> bool:
    """Up to date, or not to be had here (the wrappers then do all of it in Python)."""
    path = _torch_module_path()
    if path.exists():
        sources = (CSRC / "torch_call.cpp", PACKAGE_DIR.parent / "include" / "chord_b200.h")
        # (it holds code of torch's headers, whatever its symbols: only for the torch that it names)
        built_for = f"built for torch {_torch_version()}\0".encode()
        return path.stat().st_mtime >= max(f.stat().st_mtime for f in sources) and built_for in path.read_bytes()
    return _torch_compiler() is None


def _build_torch_module() -> None:
    """The optional ``_torch_call`` extension module (csrc/torch_call.cpp): short ways through the
    wrappers of the operators that are called once per layer and token."""
    out = _torch_module_path()
    compiler = _torch_compiler()
    reason = "no C++ compiler or no headers of Python, torch and CUDA"
    if compiler is not None:
        tmp = out.with_suffix(".tmp")
        proc = subprocess.run([*compiler[:5], str(CSRC / "torch_call.cpp"), "-o", str(tmp), *compiler[5:]],
                              capture_output=True, text=True)
        if proc.returncode == 0:
            os.replace(tmp, out)
            return
        reason = proc.stderr
    out.unlink(missing_ok=True)  # not one of another version
    warnings.warn(f"chord_b200._torch_call was not built, the wrappers take 5 to 20 us longer: {reason}")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the CUDA sources for sm_100a and link ``libchord_b200.so`` in-tree."""
    if not force and is_fresh():
        return LIB_PATH
    nvcc = _nvcc()
    obj_dir = PACKAGE_DIR / "build"
    obj_dir.mkdir(exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as pool:
        torch_module = pool.submit(_build_torch_module)
        objs = list(pool.map(lambda s: _compile(nvcc, s, obj_dir, verbose), SOURCES))
        torch_module.result()
    _build_call_module()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
