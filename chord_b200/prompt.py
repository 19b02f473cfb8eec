"""Attention of many query tokens over the paged cache: prompts and chunks of them, and batches of new tokens whose
sequences begin with a prefix that they share."""

from __future__ import annotations

import ctypes

import torch

from . import _checks, _lib
from .attention import (KVCache, _attention_scratch, _bf16_like, _cache, _ints, _locks, _queries, _scores, _sums, _table)
from .indexed_gemm import _device_index, status_word


def _offsets(name: str, x, device) -> tuple[int, int]:
    """The address of int32 offsets and how many spans they make."""
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32:
        raise TypeError(f"{name} must be a torch.int32 tensor")
    if x.ndim != 1 or x.numel() < 2:
        raise ValueError(f"{name} must be a vector of two values or more, got shape {tuple(x.shape)}")
    return _ints(name, x, x.numel(), device), x.numel() - 1


def prompt_attention(q: torch.Tensor, cache: KVCache, block_tables: torch.Tensor, lengths: torch.Tensor,
                     offsets: torch.Tensor, *, scale: float | None = None, window: int | None = None,
                     cap: float | None = None, slopes: torch.Tensor | None = None,
                     prefixes: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                     outputs: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens of ragged sequences, prompts or chunks of them, over the sequences' tokens in the cache.

    ``q`` is BF16 ``[tokens, heads, head_dim]`` (rows may be strided), sequence after sequence: those from ``offsets[b]``
    to ``offsets[b + 1]`` (int32 ``[batch + 1]``, never falling) are the last tokens of sequence ``b``, whose
    ``lengths[b]`` tokens, with their keys and values, are in the cache already.  ``cache``, ``block_tables``, ``scale``,
    ``cap`` and ``slopes`` are as for :func:`paged_attention`.  A token sees itself and those before it and

    * with ``window`` only the last so many of these;
    * with ``starts`` (int32 ``[tokens]``) none before position ``starts[t]`` of its sequence, the begin of its document;
    * with ``prefixes`` (int32 ``[batch]``) also all of its sequence's first ``prefixes[b]`` tokens, those behind it too
      (the window and the document still bound it below).

    ``slopes`` take the distance either way.  Returns BF16 ``[tokens, heads, head_dim]``; ``lse`` as for
    :func:`paged_attention`.  A token that sees nothing gives zeros and minus infinity.  Rows of tokens of no sequence
    are left as they are.  In calls that are alike in all else, the values of what a token does not see do not change its
    bits; infinities and NaN there change no more than how its weights are rounded (where neighbours see such a value, weights of
    that step are not rounded to BF16).  Other lengths, ``starts`` or ``prefixes``, of other tokens too, may change where sums are cut and
    joined, and over codes how weights are rounded.
    Offsets that fall or lie outside ``q``, lengths beyond the table and pages outside the cache are reported by
    :func:`chord_b200.check_status`; nothing outside is read or written.  The same inputs give the same bits."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None and outputs is None:
        result = direct.prompt_attention(q, cache.address, cache.index, block_tables, lengths, offsets, starts, prefixes, lse,
                                         cache.scale if scale is None else scale, window, cap, slopes)
        if result is not None:
            return result
    q_rows = _queries(q, cache)
    device, (tokens, heads) = cache.device, q.shape[:2]
    at_offsets, batch = _offsets("offsets", offsets, device)
    table = _table(block_tables, device, batch)
    at = _ints("lengths", lengths, batch, device)
    at_starts = None if starts is None else _ints("starts", starts, tokens, device)
    at_prefixes = None if prefixes is None else _ints("prefixes", prefixes, batch, device)
    scores = _scores(cache, heads, scale, window, cap, slopes)
    given = outputs is not None
    outputs = _bf16_like("outputs", outputs, q.shape, device)
    if given:
        _checks.apart("outputs", outputs, "q", q)
    sums = _sums(lse, tokens, heads, device)
    if lse is not None:
        _checks.apart("lse", lse, "q", q)
        if given:
            _checks.apart("lse", lse, "outputs", outputs)
    if tokens == 0:
        return outputs
    with _lib.on_device(device):
        size = _lib.native().chord_b200_prompt_attention_workspace_bytes(batch, tokens, heads, cache.heads, cache.head_dim)
        if size < 0:
            raise RuntimeError(_lib.last_error())
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.check(_lib.native().chord_b200_prompt_attention(
            *q_rows, cache.address, *table, at, at_offsets, at_starts, at_prefixes, outputs.data_ptr(), sums,
            workspace.data_ptr(), size, status_word(device).data_ptr(), batch, tokens, heads, ctypes.addressof(scores),
            _lib.stream_handle(device)))
    return outputs


def shared_prefix_attention(q: torch.Tensor, cache: KVCache, prefix_tables: torch.Tensor, prefix_lengths: torch.Tensor,
                            group_offsets: torch.Tensor, block_tables: torch.Tensor, lengths: torch.Tensor, *,
                            scale: float | None = None, window: int | None = None, cap: float | None = None,
                            slopes: torch.Tensor | None = None, outputs: torch.Tensor | None = None,
                            lse: torch.Tensor | None = None, locks: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`paged_attention` of one new token per sequence, for a batch in groups of neighbours that share a prefix.

    The tokens of sequence ``b`` of group ``g``, ``group_offsets[g] <= b < group_offsets[g + 1]`` (int32 ``[groups + 1]``,
    from zero to the batch, never falling), are the ``prefix_lengths[g]`` ones of ``prefix_tables[g]`` (int32 ``[groups,
    pages]``) and then its own ``lengths[b]`` ones of ``block_tables[b]``.  Either may be none.  Keys and values of a prefix
    are read once for its whole group.  The other arguments, the results and what is reported are as for
    :func:`paged_attention`, over the sequence as a whole: its window, distances and ``lse``."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None and outputs is None and locks is None:
        result = direct.shared_prefix_attention(q, cache.address, cache.index, prefix_tables, prefix_lengths, group_offsets,
                                                block_tables, lengths, lse, cache.scale if scale is None else scale, window,
                                                cap, slopes)
        if result is not None:
            return result
    q_rows = _queries(q, cache)
    device, (batch, heads) = cache.device, q.shape[:2]
    at_groups, groups = _offsets("group_offsets", group_offsets, device)
    prefix_table = _table(prefix_tables, device, groups, "prefix_tables")
    at_prefixes = _ints("prefix_lengths", prefix_lengths, groups, device)
    table = _table(block_tables, device, batch)
    at = _ints("lengths", lengths, batch, device)
    scores = _scores(cache, heads, scale, window, cap, slopes)
    given = outputs is not None
    outputs = _bf16_like("outputs", outputs, q.shape, device)
    if given:
        _checks.apart("outputs", outputs, "q", q)
    sums = _sums(lse, batch, heads, device)
    if lse is not None:
        _checks.apart("lse", lse, "q", q)
        if given:
            _checks.apart("lse", lse, "outputs", outputs)
    if batch == 0:
        return outputs
    with _lib.on_device(device):
        words, _ = _attention_scratch(_device_index(device), cache.head_dim, heads // cache.heads)
        size = _lib.native().chord_b200_shared_prefix_attention_workspace_bytes(groups, batch, heads, cache.heads, cache.head_dim)
        if size < 0:
            raise RuntimeError(_lib.last_error())
        locks = _locks(locks, words, device)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.check(_lib.native().chord_b200_shared_prefix_attention(
            *q_rows, cache.address, *prefix_table, at_prefixes, at_groups, groups, *table, at, outputs.data_ptr(), sums,
            locks.data_ptr(), locks.numel(), workspace.data_ptr(), size, status_word(device).data_ptr(), batch, heads,
            ctypes.addressof(scores), _lib.stream_handle(device)))
    return outputs


__all__ = ["prompt_attention", "shared_prefix_attention"]
