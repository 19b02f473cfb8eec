"""The attention half of a decoder layer for one new token per sequence: norms of queries and keys
with the position rotation, the paged key-value cache, and the attention over it.  The reference ends
at the expert products; a serving engine runs these steps between them."""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _checks, _lib
from .indexed_gemm import _device_index, default_locks, status_word

HEAD_DIMS = (64, 96, 128, 192, 256)  # of paged_attention


class KVCache:
    """Pages of keys and values: a handle on the caller's tensors, checked once.

    ``k`` and ``v`` are ``[pages, heads, page_size, head_dim]``: BF16, or uint8 codes with FP32 scales
    ``k_scale`` and ``v_scale`` ``[pages, heads, page_size]``, one for what a head keeps of a token:
    ``value = (code - 128) * scale`` with ``scale = max |x| / 127``.  The tensors may be views with
    any strides that leave each row of ``head_dim`` contiguous and on a 16-byte boundary, the same for
    keys and values, so pages of ``[page_size, heads, head_dim]`` work through ``transpose(1, 2)``.
    ``head_dim`` is a multiple of 16 up to 256.  :func:`kv_cache` allocates one."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_pages", "heads", "page_size", "head_dim", "device", "address",
                 "index", "scale", "_descriptor")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        coded = k_scale is not None or v_scale is not None
        for name, t in (("k", k), ("v", v)):
            _checks.tensor(name, t, dtype=torch.uint8 if coded else torch.bfloat16, ndim=4, contiguous=False, nonempty=True)
        if k.shape != v.shape or k.stride() != v.stride() or k.device != v.device:
            raise ValueError(f"k and v must be alike, got {tuple(k.shape)} with strides {k.stride()} on {k.device} and "
                             f"{tuple(v.shape)} with strides {v.stride()} on {v.device}")
        num_pages, heads, page_size, head_dim = k.shape
        if head_dim % 16 or head_dim > 256:
            raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {head_dim}")
        if num_pages * page_size >= 2**31:
            raise ValueError(f"a cache holds fewer than 2^31 tokens, got {num_pages} pages of {page_size}")
        unit = 16 // k.element_size()
        if k.stride(3) != 1 or any(s % unit for s in k.stride()[:3]) or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError(f"k and v must have contiguous rows on 16-byte boundaries, got strides {k.stride()}")
        scale_strides = (0, 0, 0)
        if coded:
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                _checks.tensor(name, t, dtype=torch.float32, ndim=3, device=k.device, contiguous=False)
                if t.shape != k.shape[:3]:
                    raise ValueError(f"{name} must have shape {tuple(k.shape[:3])}, got {tuple(t.shape)}")
            if k_scale.stride() != v_scale.stride():
                raise ValueError(f"k_scale and v_scale must have the same strides, got {k_scale.stride()} and "
                                 f"{v_scale.stride()}")
            scale_strides = k_scale.stride()
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.heads, self.page_size, self.head_dim = num_pages, heads, page_size, head_dim
        self.device, self.index, self.scale = k.device, _device_index(k.device), head_dim ** -0.5
        self._descriptor = _lib.KVCacheDescriptor(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if coded else None, v_scale.data_ptr() if coded else None,
            num_pages, page_size, heads, head_dim, *k.stride()[:3], *scale_strides)
        self.address = ctypes.addressof(self._descriptor)


def kv_cache(num_pages: int, page_size: int, heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
             device=None) -> KVCache:
    """An empty :class:`KVCache` of ``num_pages`` pages of ``page_size`` tokens; ``dtype`` BF16, or
    uint8 for codes with a scale per row."""
    for name, value in (("num_pages", num_pages), ("page_size", page_size), ("heads", heads), ("head_dim", head_dim)):
        _checks.integer(name, value, minimum=1)
    if dtype not in (torch.bfloat16, torch.uint8):
        raise TypeError(f"dtype must be torch.bfloat16 or torch.uint8, got {dtype}")
    device = torch.device("cuda") if device is None else torch.device(device)
    shape = (num_pages, heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype == torch.bfloat16:
        return KVCache(k, v)
    return KVCache(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def _cache(cache) -> KVCache:
    if not isinstance(cache, KVCache):
        raise TypeError(f"cache must be a KVCache, got {type(cache).__name__}")
    return cache


def _rows(name: str, x, device, tokens: int, heads: int | None, dim: int):
    """``x`` as BF16 ``[tokens, heads, dim]`` with rows on 16-byte boundaries: (address, token stride,
    head stride)."""
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be a torch.bfloat16 tensor")
    if x.ndim != 3 or x.shape[0] != tokens or x.shape[2] != dim or (heads is not None and x.shape[1] != heads) or not x.shape[1]:
        raise ValueError(f"{name} must have shape {(tokens, 'heads' if heads is None else heads, dim)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}, got {x.device}")
    token, head, element = x.stride()
    if element != 1 or token % 8 or head % 8 or x.data_ptr() % 16:
        raise ValueError(f"{name} must have contiguous rows on 16-byte boundaries, got strides {x.stride()}")
    return x.data_ptr(), token, head


def _ints(name: str, x, count: int, device) -> int:
    """The address of ``count`` contiguous int32 values on ``device``."""
    if (isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.ndim == 1 and x.shape[0] == count
            and x.device == device and x.is_contiguous()):
        return x.data_ptr()
    _checks.tensor(name, x, dtype=torch.int32, ndim=1, device=device)
    raise ValueError(f"{name} must hold {count} values, got {x.numel()}")


def _table(x, device, batch: int, name: str = "block_tables"):
    """A block table int32 ``[batch, pages]``: (address, row stride, pages)."""
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32:
        raise TypeError(f"{name} must be a torch.int32 tensor")
    if x.ndim != 2 or x.shape[0] != batch or x.shape[1] == 0 or x.device != device:
        raise ValueError(f"{name} must be [{batch}, pages] on {device}, got {tuple(x.shape)} on {x.device}")
    if x.stride(1) != 1 and x.shape[1] > 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    return x.data_ptr(), x.stride(0), x.shape[1]


def _bf16_like(name: str, out, shape, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=device)
    if not isinstance(out, torch.Tensor) or out.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be a torch.bfloat16 tensor")
    if tuple(out.shape) != tuple(shape) or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous BF16 {tuple(shape)} on {device} on a 16-byte boundary, got "
                         f"{tuple(out.shape)} on {out.device}")
    return out


def _rotation(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved, kv_heads):
    """The checks that qk_norm_rope and qk_norm_rope_write share: their common C arguments."""
    if not isinstance(q, torch.Tensor) or q.ndim != 3 or q.dtype is not torch.bfloat16:
        raise TypeError("q must be a 3D torch.bfloat16 tensor")
    if not q.is_cuda:
        raise ValueError(f"q must be a CUDA tensor, got device {q.device}")
    device = q.device
    _checks.supported_gpu(device)
    tokens, heads, dim = q.shape
    if dim % 16 or dim > 256 or dim == 0:
        raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {dim}")
    q_rows = _rows("q", q, device, tokens, heads, dim)
    k_rows = _rows("k", k, device, tokens, kv_heads, dim)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if not (isinstance(w, torch.Tensor) and w.dtype is torch.bfloat16 and w.shape == (dim,) and w.device == device
                and w.is_contiguous() and w.data_ptr() % 16 == 0):
            _checks.tensor(name, w, dtype=torch.bfloat16, ndim=1, device=device)
            raise ValueError(f"{name} must hold {dim} values on a 16-byte boundary, got {w.numel()}")
    if not (isinstance(cos_sin, torch.Tensor) and cos_sin.dtype is torch.float32 and cos_sin.ndim == 2
            and cos_sin.device == device and cos_sin.is_contiguous() and cos_sin.shape[0] > 0
            and cos_sin.data_ptr() % 16 == 0):
        _checks.tensor("cos_sin", cos_sin, dtype=torch.float32, ndim=2, device=device)
        raise ValueError("cos_sin must have a row for some position and lie on a 16-byte boundary")
    rotary = cos_sin.shape[1]
    if rotary % 16 or rotary > dim:
        raise ValueError(f"cos_sin must have a multiple of 16 up to head_dim={dim} columns, got {rotary}")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0 <= eps < math.inf:
        raise ValueError(f"eps must be a finite number of at least zero, got {eps!r}")
    _checks.flag("interleaved", interleaved)
    at = _ints("positions", positions, tokens, device)
    return (device, tokens, heads, dim, q_rows, k_rows,
            (q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], rotary, int(interleaved), at))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 cos_sin: torch.Tensor, positions: torch.Tensor, *, eps: float = 1e-6, interleaved: bool = False,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Root-mean-square norms of each head's queries and keys and the position rotation, in one pass, in FP32
    (squares too: finite elements of 2^60 or more may count as infinite).

    ``q`` is BF16 ``[tokens, heads, head_dim]`` and ``k`` ``[tokens, kv_heads, head_dim]``; both may be
    views of the fused projection's result.  ``q_weight`` and ``k_weight`` are BF16 ``[head_dim]``.
    ``cos_sin`` is FP32 ``[max_positions, rotary_dim]``, cosines and then sines of each position's
    angles; the first ``rotary_dim`` elements of a head turn (a multiple of 16, none with zero
    columns), element ``i`` with ``i + rotary_dim / 2`` or, ``interleaved``, ``2 i`` with ``2 i + 1``.
    ``positions`` is int32 ``[tokens]``; a position outside the table gives zeros and is reported by
    :func:`chord_b200.check_status`.  Returns BF16 ``(q_out, k_out)``, contiguous; contiguous inputs may be
    given as their own outputs, and outputs overlap nothing else of the call."""
    direct = _lib.direct()
    if direct is not None and q_out is None and k_out is None:
        result = direct.qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved)
        if result is not None:
            return result
    device, tokens, heads, dim, q_rows, k_rows, rest = _rotation(q, k, q_weight, k_weight, cos_sin, positions, eps,
                                                                 interleaved, None)
    given = q_out is not None or k_out is not None
    q_out = _bf16_like("q_out", q_out, q.shape, device)
    k_out = _bf16_like("k_out", k_out, k.shape, device)
    if given:
        _checks.apart("q_out", q_out, "q", q, in_place=True)
        _checks.apart("k_out", k_out, "k", k, in_place=True)
        for name, out, other_name, other in (("q_out", q_out, "k", k), ("k_out", k_out, "q", q), ("q_out", q_out, "k_out", k_out)):
            _checks.apart(name, out, other_name, other)
    with _lib.on_device(device):
        _lib.check(_lib.native().chord_b200_qk_norm_rope(
            *q_rows, *k_rows, *rest, q_out.data_ptr(), k_out.data_ptr(), tokens, heads, k.shape[1], dim,
            status_word(device).data_ptr(), eps, _lib.stream_handle(device)))
    return q_out, k_out


def qk_norm_rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor,
                       k_weight: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor, cache: KVCache,
                       slots: torch.Tensor, *, eps: float = 1e-6, interleaved: bool = False,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`qk_norm_rope` whose keys go, with the values as they are, straight into the cache: token
    ``t`` at slot ``slots[t]`` (int32, page * page_size + place; negative: not kept).  The slots that are kept are
    distinct, as for :func:`cache_write`.  Keys are quantised from FP32.  Returns the queries."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None and q_out is None:
        result = direct.qk_norm_rope_write(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved, v,
                                           cache.address, cache.index, slots)
        if result is not None:
            return result
    device, tokens, heads, dim, q_rows, k_rows, rest = _rotation(q, k, q_weight, k_weight, cos_sin, positions, eps,
                                                                 interleaved, cache.heads)
    if dim != cache.head_dim or device != cache.device:
        raise ValueError(f"q and k have head_dim={dim} on {device}, the cache {cache.head_dim} on {cache.device}")
    v_rows = _rows("v", v, device, tokens, cache.heads, dim)
    at = _ints("slots", slots, tokens, device)
    given = q_out is not None
    q_out = _bf16_like("q_out", q_out, q.shape, device)
    if given:
        _checks.apart("q_out", q_out, "q", q, in_place=True)
        for name, other in (("k", k), ("v", v)):
            _checks.apart("q_out", q_out, name, other)
    with _lib.on_device(device):
        _lib.check(_lib.native().chord_b200_qk_norm_rope_write(
            *q_rows, *k_rows, *v_rows, *rest, q_out.data_ptr(), cache.address, at, tokens, heads,
            status_word(device).data_ptr(), eps, _lib.stream_handle(device)))
    return q_out


def cache_write(k: torch.Tensor, v: torch.Tensor, cache: KVCache, slots: torch.Tensor) -> None:
    """Keys and values, BF16 ``[tokens, kv_heads, head_dim]``, into the cache: token ``t`` at slot
    ``slots[t]`` (int32, page * page_size + place; negative: not kept).  The slots that are kept are distinct: a row
    that two tokens of a call name holds parts of either.  A slot outside the cache is not written and is reported by :func:`chord_b200.check_status`.  A row that holds an infinity or a
    NaN reads back as NaN from an 8-bit cache."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None and direct.cache_write(k, v, cache.address, cache.index, slots):
        return
    device = cache.device
    if not isinstance(k, torch.Tensor) or k.ndim != 3:
        raise TypeError("k must be a 3D torch.bfloat16 tensor")
    _checks.supported_gpu(device)
    tokens = k.shape[0]
    k_rows = _rows("k", k, device, tokens, cache.heads, cache.head_dim)
    v_rows = _rows("v", v, device, tokens, cache.heads, cache.head_dim)
    at = _ints("slots", slots, tokens, device)
    with _lib.on_device(device):
        _lib.check(_lib.native().chord_b200_cache_write(
            *k_rows, *v_rows, cache.address, at, tokens, status_word(device).data_ptr(), _lib.stream_handle(device)))


def cache_read(cache: KVCache, block_tables: torch.Tensor, offsets: torch.Tensor, total: int, *,
               k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
    """The keys and values of whole sequences out of the cache as BF16 ``[total, kv_heads, head_dim]``,
    one sequence after another: sequence ``b`` fills rows ``offsets[b]`` to ``offsets[b + 1]`` with its
    first tokens.  ``block_tables`` is int32 ``[batch, pages]``, ``offsets`` int32 ``[batch + 1]`` and
    never falls; rows of no sequence are zeros, as are tokens whose page the table or the cache does
    not have, which :func:`chord_b200.check_status` reports."""
    _cache(cache)
    direct = _lib.direct()
    if direct is not None and k_out is None and v_out is None:
        result = direct.cache_read(cache.address, cache.index, block_tables, offsets, total)
        if result is not None:
            return result
    device = cache.device
    _checks.supported_gpu(device)
    _checks.integer("total", total, minimum=0)
    if not isinstance(offsets, torch.Tensor) or offsets.ndim != 1 or offsets.numel() < 2:
        raise ValueError("offsets must be a vector of batch + 1 values")
    batch = offsets.numel() - 1
    at = _ints("offsets", offsets, batch + 1, device)
    table = _table(block_tables, device, batch)
    shape = (total, cache.heads, cache.head_dim)
    given = k_out is not None and v_out is not None
    k_out, v_out = _bf16_like("k_out", k_out, shape, device), _bf16_like("v_out", v_out, shape, device)
    if given:
        _checks.apart("k_out", k_out, "v_out", v_out)
    with _lib.on_device(device):
        _lib.check(_lib.native().chord_b200_cache_read(
            cache.address, *table, at, batch, k_out.data_ptr(), v_out.data_ptr(), total,
            status_word(device).data_ptr(), _lib.stream_handle(device)))
    return k_out, v_out


def _scores(cache: KVCache, heads: int, scale, window, cap, slopes) -> _lib.ScoresDescriptor:
    """The checks of what shapes scores: their C form."""
    if scale is None:
        scale = cache.scale
    elif isinstance(scale, bool) or not isinstance(scale, (int, float)) or not math.isfinite(scale):
        raise ValueError(f"scale must be a finite number, got {scale!r}")
    if window is None:
        window = 0
    else:
        _checks.integer("window", window, minimum=1)
        if window >= 2**31:
            raise ValueError(f"window must be below 2^31, got {window}")
    if cap is None:
        cap = 0.0
    elif isinstance(cap, bool) or not isinstance(cap, (int, float)) or not 1e-30 <= cap <= 1e30:
        raise ValueError(f"cap must be a number from 1e-30 to 1e30, got {cap!r}")
    address = None
    if slopes is not None:
        if not (isinstance(slopes, torch.Tensor) and slopes.dtype is torch.float32 and slopes.shape == (heads,)
                and slopes.device == cache.device and slopes.is_contiguous()):
            _checks.tensor("slopes", slopes, dtype=torch.float32, ndim=1, device=cache.device)
            raise ValueError(f"slopes must hold {heads} values, got {slopes.numel()}")
        address = slopes.data_ptr()
    return _lib.ScoresDescriptor(scale, cap, address, window)


def _sums(lse, tokens: int, heads: int, device) -> int | None:
    """The address of FP32 ``[tokens, heads]``, if given."""
    if lse is None:
        return None
    if not (isinstance(lse, torch.Tensor) and lse.dtype is torch.float32 and lse.shape == (tokens, heads)
            and lse.device == device and lse.is_contiguous()):
        _checks.tensor("lse", lse, dtype=torch.float32, ndim=2, device=device)
        raise ValueError(f"lse must have shape {(tokens, heads)}, got {tuple(lse.shape)}")
    return lse.data_ptr()


def _queries(q, cache: KVCache):
    """``q`` as BF16 ``[tokens, heads, head_dim]`` over ``cache``: (address, token stride, head stride)."""
    if not isinstance(q, torch.Tensor) or q.ndim != 3 or q.dtype is not torch.bfloat16:
        raise TypeError("q must be a 3D torch.bfloat16 tensor")
    _checks.supported_gpu(cache.device)
    rows = _rows("q", q, cache.device, q.shape[0], None, cache.head_dim)
    if cache.head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {cache.head_dim}")
    if q.shape[1] % cache.heads:
        raise ValueError(f"the number of query heads must be a multiple of the cache's {cache.heads}, got {q.shape[1]}")
    return rows


def _locks(locks, words: int, device) -> torch.Tensor:
    if locks is None:
        return default_locks(device)
    _checks.tensor("locks", locks, dtype=torch.int32, ndim=1, device=device)
    if locks.numel() < words:
        raise RuntimeError(f"locks has {locks.numel()} lock words, this launch needs at least {words}")
    return locks


@functools.lru_cache(maxsize=64)
def _attention_scratch(device_index: int, head_dim: int, group: int):
    """(lock words, workspace bytes), asked of the library once per device and shape."""
    del device_index  # a cache key only (the current device must be it)
    lib = _lib.load()
    words = lib.chord_b200_paged_attention_lock_words()
    size = lib.chord_b200_paged_attention_workspace_bytes(head_dim, group)
    if words < 0 or size < 0:
        raise RuntimeError(_lib.last_error())
    return words, size


def paged_attention(q: torch.Tensor, cache: KVCache, block_tables: torch.Tensor, lengths: torch.Tensor, *,
                    scale: float | None = None, window: int | None = None, cap: float | None = None,
                    slopes: torch.Tensor | None = None, outputs: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None, locks: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its tokens in the cache.

    ``q`` is BF16 ``[batch, heads, head_dim]`` (rows may be strided), ``heads`` a multiple of the
    cache's: head ``h`` reads key-value head ``h // (heads // cache.heads)``.  ``head_dim`` is 64, 96,
    128, 192 or 256.  ``block_tables`` int32 ``[batch, pages]`` and ``lengths`` int32 ``[batch]`` say
    where each sequence's tokens are; the new token's own key and value are the last of them if they
    are written first.  ``window`` keeps the last so many tokens.  ``scale`` is ``head_dim ** -0.5``
    where it is not given.  With ``cap`` scores become ``cap * tanh(score / cap)``; with ``slopes`` (FP32 ``[heads]``)
    ``slopes[h]`` times a token's distance to the new one is then taken off.  Returns BF16 ``[batch, heads, head_dim]``
    (``outputs``, where given, must not overlap ``q``); ``lse``, if given, FP32 ``[batch,
    heads]``, receives the logarithm of each softmax's sum, with which results over parts of a
    sequence can be joined, and overlaps neither ``q`` nor ``outputs``.  A sequence of length zero gives zeros and minus infinity; a head whose query
    holds an infinity gives NaN over an 8-bit cache.

    Page ids outside the cache count as keys and values of zero and, like lengths beyond the
    table, are reported by :func:`chord_b200.check_status`.  ``locks`` is as for ``indexed``: zeroed
    int32, left zeroed, one buffer per launches that may overlap; with ``None`` a per-stream buffer of
    the library's.  The same inputs give the same bits."""
    _cache(cache)
    shaped = cap is not None or slopes is not None
    direct = _lib.direct()
    if direct is not None and outputs is None and locks is None and window != 0:
        if shaped:
            result = direct.paged_attention_shaped(q, cache.address, cache.index, block_tables, lengths, lse,
                                                   cache.scale if scale is None else scale, window, cap, slopes)
        else:
            result = direct.paged_attention(q, cache.address, cache.index, block_tables, lengths, lse,
                                            0 if window is None else window, cache.scale if scale is None else scale)
        if result is not None:
            return result
    q_rows = _queries(q, cache)
    device, dim, (batch, heads) = cache.device, cache.head_dim, q.shape[:2]
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
        words, size = _attention_scratch(_device_index(device), dim, heads // cache.heads)
        locks = _locks(locks, words, device)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        rest = (outputs.data_ptr(), sums, locks.data_ptr(), locks.numel(), workspace.data_ptr(), size,
                status_word(device).data_ptr(), batch, heads)
        stream = _lib.stream_handle(device)
        if shaped:
            _lib.check(_lib.native().chord_b200_paged_attention_shaped(*q_rows, cache.address, *table, at, *rest,
                                                                       ctypes.addressof(scores), stream))
        else:
            _lib.check(_lib.native().chord_b200_paged_attention(*q_rows, cache.address, *table, at, *rest, scores.window,
                                                                scores.scale, stream))
    return outputs


__all__ = ["KVCache", "kv_cache", "cache_read", "cache_write", "paged_attention", "qk_norm_rope", "qk_norm_rope_write"]
