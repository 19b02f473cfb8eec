"""The short ways through the wrappers run while other threads of the interpreter run: entry points that take
their time, in place of the library's, do not stop them."""

import ctypes
import shutil
import subprocess
import threading
import time

import pytest
import torch

import chord_b200
from chord_b200 import _lib, indexed_gemm
from tests.cases import make_weights

pytestmark = pytest.mark.gpu

SLOW = r"""
#include <stdint.h>
#include <unistd.h>
static int slow(void) { usleep(300000); return 1; }   /* (refused: nothing has been written) */
int slow_call() { return slow(); }
int64_t small_size(int64_t a, int64_t b) { return 1024 + 0 * (a + b); }
"""


@pytest.fixture
def slow_entries(device, tmp_path):
    module = _lib.direct()
    if module is None or shutil.which("gcc") is None:
        pytest.skip("the module was not built")
    indexed_gemm.status_word(device)
    indexed_gemm.default_locks(device)
    (tmp_path / "slow.c").write_text(SLOW)
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "slow.c"), "-o", str(tmp_path / "slow.so")], check=True)
    slow = ctypes.CDLL(str(tmp_path / "slow.so"))
    at = [ctypes.cast(f, ctypes.c_void_p).value for f in [slow.slow_call] * 6 + [slow.small_size]]
    module.entries(*at)
    yield module
    _lib.direct.cache_clear()
    assert _lib.direct() is module   # (with the library's entry points again)


def test_other_threads_run(device, slow_entries):
    module = slow_entries
    codes, scale = make_weights(1, 128, 64, 5)
    w = chord_b200.pack_w4a16(codes.to(device), scale.to(device))
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device=device)
    cache = chord_b200.kv_cache(2, 4, 2, 64, device=device)
    heads = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=device)
    kv = heads[:, :2]
    weight, angles = torch.ones(64, dtype=torch.bfloat16, device=device), torch.zeros((8, 64), device=device)
    ints = torch.zeros(2, dtype=torch.int32, device=device)
    table = torch.zeros((2, 2), dtype=torch.int32, device=device)
    offsets = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    calls = {
        "gemv": (x, w.packed, w.scale, 128, 64, 1, None, 1, 0),
        "qk_norm_rope": (heads, kv, weight, weight, angles, ints, 1e-6, False),
        "qk_norm_rope_write": (heads, kv, weight, weight, angles, ints, 1e-6, False, kv, cache.address, cache.index, ints),
        "cache_write": (kv, kv, cache.address, cache.index, ints),
        "cache_read": (cache.address, cache.index, table, offsets, 2),
        "paged_attention": (heads, cache.address, cache.index, table, ints, None, 0, 0.125),
    }
    for name, arguments in calls.items():
        turns, stop = [], threading.Event()

        def count():
            while not stop.is_set():
                turns.append(time.perf_counter())
                time.sleep(0.005)

        thread = threading.Thread(target=count)
        thread.start()
        time.sleep(0.02)
        begin = time.perf_counter()
        assert getattr(module, name)(*arguments) is None
        end = time.perf_counter()
        stop.set()
        thread.join()
        assert end - begin > 0.25, name
        assert sum(begin + 0.05 < t < end - 0.05 for t in turns) > 5, name
