"""Bounds on the paged cache: what its tokens get of the attention, and eviction of those that get least."""

from __future__ import annotations

import ctypes

import torch

from . import _checks, _lib
from .attention import KVCache, _cache, _ints, _queries, _scores, _sums, _table
from .indexed_gemm import status_word


def _weights(name: str, x, batch: int, heads: int, device) -> tuple[int, int, int, int]:
    """FP32 ``[batch, heads, width]`` with contiguous rows: (address, batch stride, head stride, width)."""
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.float32:
        raise TypeError(f"{name} must be a torch.float32 tensor")
    if x.ndim != 3 or x.shape[0] != batch or x.shape[1] != heads or x.shape[2] == 0 or x.device != device:
        raise ValueError(f"{name} must be [{batch}, {heads}, width] on {device}, got {tuple(x.shape)} on {x.device}")
    if x.stride(2) != 1 and x.shape[2] > 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    return x.data_ptr(), x.stride(0), x.stride(1), x.shape[2]


def attention_weights(q: torch.Tensor, cache: KVCache, block_tables: torch.Tensor, lengths: torch.Tensor,
                      lse: torch.Tensor, *, scale: float | None = None, window: int | None = None,
                      cap: float | None = None, slopes: torch.Tensor | None = None,
                      weights: torch.Tensor | None = None) -> torch.Tensor:
    """What each token of the cache got of the new tokens' attention: FP32 ``[batch, cache.heads, width]``, for every
    sequence and key-value head the softmax weights of its tokens, summed over the query heads that share the head.

    The arguments are those of the :func:`paged_attention` call that gave ``lse``.  Without ``weights`` the result is new,
    as wide as the table, with zeros for tokens that are not seen; with it (FP32, as wide as the longest sequence or
    wider, rows contiguous and apart from each other, ``q`` and ``lse``) they are added to it, token by token, and it is returned.  The same inputs give the same bits.
    What :func:`paged_attention` reports is reported, and lengths beyond ``weights``."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None:
        result = direct.attention_weights(q, cache.address, cache.index, block_tables, lengths, lse, weights,
                                          cache.scale if scale is None else scale, window, cap, slopes)
        if result is not None:
            return result
    q_rows = _queries(q, cache)
    device, (batch, heads) = cache.device, q.shape[:2]
    table = _table(block_tables, device, batch)
    at = _ints("lengths", lengths, batch, device)
    if lse is None:
        raise TypeError("lse must be a torch.Tensor")
    sums = _sums(lse, batch, heads, device)
    scores = _scores(cache, heads, scale, window, cap, slopes)
    if batch > 65535:
        raise ValueError(f"the batch must be at most 65535, got {batch}")
    add = weights is not None
    if not add:
        weights = torch.empty((batch, cache.heads, table[2] * cache.page_size), dtype=torch.float32, device=device)
    *to, width = _weights("weights", weights, batch, cache.heads, device) if batch else (0, 0, 0, 0)
    if add and batch:
        (inner, rows), (outer, others) = sorted(zip(weights.stride()[:2], weights.shape[:2]))
        if (rows > 1 and inner < width) or (others > 1 and outer < (rows - 1) * inner + width):
            raise ValueError(f"rows of weights must not overlap, got strides {weights.stride()}")
        extent = weights.as_strided((sum((n - 1) * s for n, s in zip(weights.shape, weights.stride())) + 1,), (1,))
        _checks.apart("weights", extent, "lse", lse)
        _checks.apart("weights", extent, "q", q)
    if batch == 0:
        return weights
    with _lib.on_device(device):
        _lib.check(_lib.native().chord_b200_attention_weights(
            *q_rows, cache.address, *table, at, sums, *to, width, int(add), status_word(device).data_ptr(), batch, heads,
            ctypes.addressof(scores), _lib.stream_handle(device)))
    return weights


def cache_evict(cache: KVCache, block_tables: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, keep: int, *,
                first: int = 0, recent: int = 0, new_tables: torch.Tensor | None = None):
    """Cuts sequences down to their ``keep`` tokens that matter, each key-value head on its own.

    A head keeps its first ``first`` tokens, its last ``recent`` ones and, of those between, the ones with the largest
    ``weights`` (FP32 ``[batch, cache.heads, width]``, as :func:`attention_weights` gathers them; equal ones from the first
    on, NaN counts as the largest), ``keep`` in all and in order; a sequence that has no more keeps them all.  The rows move to
    the front of the sequence's pages or, with ``new_tables`` (int32 ``[batch, pages]``), into those, which are no pages of
    ``block_tables``; two sequences share no page that is written.  Rows behind the kept ones stay as they are.  Keys
    keep the positions that they were turned by; windows and distances count the kept tokens.

    Returns the new lengths, int32 ``[batch]``, and the kept tokens' weights, FP32 ``[batch, cache.heads, width]`` (``keep``
    wide, if that is more), zeros behind them.  Lengths beyond the table or the weights and pages outside the cache are
    reported by :func:`chord_b200.check_status`."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None:
        result = direct.cache_evict(cache.address, cache.index, block_tables, lengths, weights, keep, first, recent, new_tables)
        if result is not None:
            return result
    device = cache.device
    _checks.supported_gpu(device)
    if not isinstance(lengths, torch.Tensor) or lengths.ndim != 1:
        raise TypeError("lengths must be a vector of torch.int32")
    batch = lengths.numel()
    at = _ints("lengths", lengths, batch, device)
    table = _table(block_tables, device, batch)
    new_table = (None, 0, 0) if new_tables is None else _table(new_tables, device, batch, "new_tables")
    *held, width = _weights("weights", weights, batch, cache.heads, device)
    _checks.integer("keep", keep, minimum=1)
    if keep >= 2**28:
        raise ValueError(f"keep must be below 2^28, got {keep}")
    _checks.integer("first", first, minimum=0)
    _checks.integer("recent", recent, minimum=0)
    if first + recent > keep:
        raise ValueError(f"first and recent must not be more than keep={keep} together, got {first} and {recent}")
    if new_tables is not None and new_tables.shape[1] * cache.page_size < min(keep, width, block_tables.shape[1] * cache.page_size):
        raise ValueError(f"new_tables must have room for {min(keep, width)} tokens, got {new_tables.shape[1]} pages of {cache.page_size}")
    if batch > 65535:
        raise ValueError(f"the batch must be at most 65535, got {batch}")
    new_lengths = torch.empty((batch,), dtype=torch.int32, device=device)
    new_weights = torch.empty((batch, cache.heads, max(width, keep)), dtype=torch.float32, device=device)
    if batch == 0:
        return new_lengths, new_weights
    with _lib.on_device(device):
        size = batch * cache.heads * min(keep, width) * 4
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.check(_lib.native().chord_b200_cache_evict(
            cache.address, *table, *new_table, at, *held, width, new_lengths.data_ptr(), new_weights.data_ptr(),
            new_weights.shape[2], workspace.data_ptr(), size, status_word(device).data_ptr(), batch, keep, first, recent,
            _lib.stream_handle(device)))
    return new_lengths, new_weights


__all__ = ["attention_weights", "cache_evict"]
