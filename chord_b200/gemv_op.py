"""``gemv``: products of a few rows with packed 4-bit weights, without routing blocks.  No
counterpart in the reference, whose operators take their rows by routing blocks (``indexed``) or by
groups (``contiguous``, ``masked``)."""

from __future__ import annotations

import torch

from . import _checks, _lib
from .indexed_gemm import status_word
from .packing import PreparedWeight

MAX_ROWS = 16           # rows that share one weight
MAX_ROUTED_ROWS = 65535  # rows with an expert each


def gemv(x: torch.Tensor, weight: PreparedWeight, *, expert_ids: torch.Tensor | None = None, top_k: int = 1,
         expert_base: int = 0, outputs: torch.Tensor | None = None) -> torch.Tensor:
    """BF16 ``x [M, K]`` times a weight from ``pack_w4a16``, for single tokens and small batches.

    Without ``expert_ids`` the weight holds one expert (a dense layer: an attention projection, a
    shared expert) and ``M`` is at most 16; returns BF16 ``[M, N]``.  More rows: ``indexed``,
    ``contiguous`` or ``masked``.

    With ``expert_ids`` (int32, ``M * top_k`` values in any shape, token after token, as a router
    leaves them) row ``r`` of the result is ``x[r // top_k]`` times the weight of expert
    ``expert_ids[r] - expert_base``; rows of experts that the weight does not hold are zero.  Returns
    BF16 ``[M * top_k, N]``.  Every row reads a weight of its own, so this is the form for a few
    tokens; from about a dozen on ``moe_align_block_size`` and ``indexed`` read shared experts once.
    For the down projection pass the routed activations and ``top_k=1``.

    The rows of ``x`` may be a view with a row stride; ``outputs`` must not overlap it.  Weights are ``(code - 8) * scale`` without a
    rounding to BF16; sums are FP32, the result is rounded once.
    """
    direct = _lib.direct()
    if direct is not None and outputs is None and type(weight) is PreparedWeight:
        result = direct.gemv(x, weight.packed, weight.scale, weight.n, weight.k, weight.num_experts, expert_ids, top_k,
                             expert_base)
        if result is not None:
            return result
    if not isinstance(x, torch.Tensor) or x.ndim != 2 or x.dtype != torch.bfloat16:
        raise TypeError("x must be a 2D torch.bfloat16 tensor")
    if not x.is_cuda:
        raise ValueError(f"x must be a CUDA tensor, got device {x.device}")
    device = x.device
    _checks.supported_gpu(device)
    packed, scale, num_experts, shape_n, shape_k = _checks.prepared_weight(weight, device)
    rows, k = x.shape
    if k != shape_k:
        raise ValueError(f"x K={k} does not match the weight's K={shape_k}")
    stride = x.stride(0) if rows > 1 else k
    if x.stride(1) != 1 or stride < k or stride % 2 or x.data_ptr() % 4:
        raise ValueError("x must have contiguous rows on 4-byte boundaries that do not overlap, got strides "
                         f"{tuple(x.stride())}")
    _checks.integer("top_k", top_k, minimum=1)
    _checks.integer("expert_base", expert_base, minimum=0)
    if expert_ids is None:
        if num_experts != 1:
            raise ValueError(f"a weight of {num_experts} experts needs expert_ids")
        if top_k != 1 or expert_base != 0:
            raise ValueError("top_k and expert_base go with expert_ids")
        if rows > MAX_ROWS:
            raise ValueError(f"gemv takes at most {MAX_ROWS} rows of x, got {rows}; see indexed, contiguous, masked")
        ids = None
    else:
        _checks.tensor("expert_ids", expert_ids, dtype=torch.int32, device=device)
        rows *= top_k
        if expert_ids.numel() != rows:
            raise ValueError(f"expert_ids must hold {rows} values (rows of x times top_k), got {expert_ids.numel()}")
        if rows > MAX_ROUTED_ROWS:
            raise ValueError(f"gemv takes at most {MAX_ROUTED_ROWS} routed rows, got {rows}")
        ids = expert_ids.data_ptr()
    if outputs is None:
        outputs = torch.empty((rows, shape_n), dtype=torch.bfloat16, device=device)
    else:
        _checks.bf16_output(outputs, (rows, shape_n), device, exact_shape=True)
        _checks.apart("outputs", outputs, "x", x)
    if rows == 0:
        return outputs
    if not torch.cuda.is_current_stream_capturing():
        status_word(device)  # (the kernel has no use for it; the short way above goes to devices that have one)
    with _lib.on_device(device):
        _lib.check(_lib.native().chord_b200_gemv(
            x.data_ptr(), stride, packed.data_ptr(), scale.data_ptr(), ids, outputs.data_ptr(), rows, shape_n,
            shape_k, num_experts, top_k, expert_base, _lib.stream_handle(device)))
    return outputs


__all__ = ["gemv"]
