"""chord_b200: W4A16 MoE expert GEMMs for NVIDIA B200 (sm_100a).

Drop-in for the public surface of the reference's ``chord_kernels`` package
(chord_kernels/__init__.py:6-21): ``pack_w4a16``, ``indexed``,
``indexed_block_m``, ``contiguous``, ``masked``.  Names resolve on first access,
so importing the package does not import torch.
"""

from importlib import import_module
from typing import Any

__all__ = [
    "contiguous",
    "indexed",
    "indexed_block_m",
    "masked",
    "pack_w4a16",
]

_EXPORTS = {
    "indexed": "chord_b200.indexed_gemm",
    "indexed_block_m": "chord_b200.indexed_gemm",
    "masked": "chord_b200.grouped_gemm",
    "contiguous": "chord_b200.grouped_gemm",
    "pack_w4a16": "chord_b200.packing",
    "PreparedWeight": "chord_b200.packing",
    "silu_mul": "chord_b200.fused_ops",
    "moe_align_block_size": "chord_b200.fused_ops",
    "check_status": "chord_b200.indexed_gemm",
    "indexed_gate_up_silu": "chord_b200.indexed_gemm",
    "set_option": "chord_b200._lib",
    "gemv": "chord_b200.gemv_op",
    "KVCache": "chord_b200.attention",
    "kv_cache": "chord_b200.attention",
    "cache_read": "chord_b200.attention",
    "cache_write": "chord_b200.attention",
    "paged_attention": "chord_b200.attention",
    "qk_norm_rope": "chord_b200.attention",
    "qk_norm_rope_write": "chord_b200.attention",
}


def __getattr__(name: str) -> Any:
    if name in _EXPORTS:
        value = getattr(import_module(_EXPORTS[name]), name)
        globals()[name] = value
        return value
    if f"{__name__}.{name}" in _EXPORTS.values():  # a module that no name has brought in yet
        return import_module(f"{__name__}.{name}")
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__() -> list[str]:
    return sorted(set(globals()) | set(__all__))
