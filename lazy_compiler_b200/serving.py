"""Serving operators: attention of prompts and of single new tokens, and the paged key-value cache between them.

The functions take torch tensors on one CUDA device and launch the library's kernels (``include/lazyb200.h``,
"serving") on the tensors' device, on its current stream or on ``stream``:

* :func:`window_attention` — a prompt, or the next chunk of one, over its keys: causal, optionally with a sliding
  window and a few first tokens ("sinks") that stay visible;
* :func:`paged_decode` — one new token per sequence over the pages of its keys and values;
* :func:`cache_extend`, :func:`cache_write`, :func:`cache_fork`, :func:`cache_release`, :func:`cache_trim`,
  :func:`cache_compact`, :func:`cache_copy` — the pages themselves.

A cache is a ``pool[planes, pages, kv_heads, page_size, head_dim]`` (a plane is the keys or the values of one layer)
and its :class:`CacheMaps`, int32 tensors on the device.  What is free is read from ``refs`` alone, so no operation
needs the host: a decode step can be captured in a CUDA graph.  Operations on maps return new ones, or write ``into``
given ones, which may be the same (not for :func:`cache_fork`).  :class:`PagedCache` keeps a pool with its maps.

A tensor used on another stream than the one it was made on needs ``record_stream`` or an event, as any torch tensor.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import runtime

_DTYPES = {torch.float16: runtime.LC_F16, torch.bfloat16: runtime.LC_BF16}


class CacheMaps(NamedTuple):
    """Whose pages are whose: ``table[slots, width]`` (a sequence's pages in order, -1 where there is none),
    ``lens[slots]`` (its tokens), ``refs[pages]`` (how many sequences hold the page) and, from the operation that
    made them, ``status[2]``: 0, -1 (an argument out of range) or the number of pages missing, where it is not 0 the
    maps are unchanged; and the pages free."""
    table: torch.Tensor
    lens: torch.Tensor
    refs: torch.Tensor
    status: torch.Tensor | None = None


def _stream(stream, device) -> int:
    return stream if stream is not None else torch.cuda.current_stream(device).cuda_stream


def _call(name: str, device, *args) -> None:
    """Calls the entry point with ``device`` current."""
    if device.index == torch.cuda.current_device():
        runtime.call(name, *args)
    else:
        with torch.cuda.device(device):
            runtime.call(name, *args)


def _check(t: torch.Tensor, what: str, device, dtype, shape: tuple) -> None:
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: {t.dtype} on {t.device}, expected {dtype} on {device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {shape}")


def _check_ints(t: torch.Tensor, what: str, device, shape: tuple) -> None:
    _check(t, what, device, torch.int32, shape)
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")


def _attention_dtype(q: torch.Tensor, what: str) -> int:
    if q.dtype not in _DTYPES:
        raise ValueError(f"{what}: {q.dtype} is not float16 or bfloat16")
    if not q.is_cuda:
        raise ValueError(f"{what}: on {q.device}, the kernels run on CUDA devices only")
    return _DTYPES[q.dtype]


def _inner(t: torch.Tensor, what: str) -> None:
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")


def _scale(scale, d: int) -> float:
    return 1.0 / math.sqrt(d) if scale is None else float(scale)


def window_attention(q, k, v, *, window: int = 0, sinks: int = 0, scale: float | None = None, q_lens=None, kv_lens=None,
                     out=None, return_lse: bool = False, stream: int | None = None):
    """Causal attention of ``q[batch, s_q, q_heads, d]`` over ``k, v[batch, s_kv, kv_heads, d]`` (f16 or bf16).

    Sequence ``b`` has ``q_lens[b]`` queries and ``kv_lens[b]`` keys (int32 on the device; all of them by default);
    its query ``i`` is at position ``p = kv_lens[b] - q_lens[b] + i`` and sees key ``j <= p`` when ``window`` is 0,
    ``j > p - window`` or ``j < sinks``.  ``scale`` is ``1 / sqrt(d)`` by default.  Returns ``o`` like ``q`` (``out``
    where given), with ``return_lse`` also the log-sum-exp of the scaled scores, f32 ``[batch, q_heads, s_q]``.  Rows
    that see nothing, and rows from ``q_lens[b]`` on, are 0 and -inf.  Any strides with a contiguous last axis.
    """
    dtype = _attention_dtype(q, "q")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q and k have 4 axes, got {q.dim()} and {k.dim()}")
    batch, s_q, q_heads, d = q.shape
    s_kv, kv_heads = k.shape[1], k.shape[2]
    dev = q.device
    _check(k, "k", dev, q.dtype, (batch, s_kv, kv_heads, d))
    _check(v, "v", dev, q.dtype, (batch, s_kv, kv_heads, d))
    if out is None:
        out = torch.empty((batch, s_q, q_heads, d), dtype=q.dtype, device=dev)
    else:
        _check(out, "out", dev, q.dtype, (batch, s_q, q_heads, d))
    for t, what in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        _inner(t, what)
    for t, what in ((q_lens, "q_lens"), (kv_lens, "kv_lens")):
        if t is not None:
            _check_ints(t, what, dev, (batch,))
    lse = torch.empty((batch, q_heads, s_q), dtype=torch.float32, device=dev) if return_lse else None
    strides = (ctypes.c_int64 * 12)(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3])
    _call("lc_window_attention", dev, dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
          lse.data_ptr() if return_lse else None, q_lens.data_ptr() if q_lens is not None else None,
          kv_lens.data_ptr() if kv_lens is not None else None, batch, s_q, s_kv, q_heads, kv_heads, d, strides, window,
          sinks, _scale(scale, d), _stream(stream, dev))
    return (out, lse) if return_lse else out


def paged_decode(q, k_pages, v_pages, table, lens, *, window: int = 0, sinks: int = 0, scale: float | None = None, out=None,
                 return_lse: bool = False, stream: int | None = None):
    """Attention of one new token per sequence, ``q[slots, q_heads, d]``, over its cached keys and values.

    ``k_pages, v_pages[pages, kv_heads, page_size, d]`` (a pool's planes), ``table[slots, width]`` and ``lens[slots]``
    as in :class:`CacheMaps`; ``lens`` counts the new token, whose key and value are in the cache already.  The rest
    is as in :func:`window_attention`, of which this is the single-token form; the log-sum-exp is ``[slots, q_heads]``.
    """
    dtype = _attention_dtype(q, "q")
    if q.dim() != 3 or k_pages.dim() != 4 or table.dim() != 2:
        raise ValueError(f"q, k_pages and table have 3, 4 and 2 axes, got {q.dim()}, {k_pages.dim()} and {table.dim()}")
    slots, q_heads, d = q.shape
    pages, kv_heads, page_size, _ = k_pages.shape
    dev = q.device
    _check(k_pages, "k_pages", dev, q.dtype, (pages, kv_heads, page_size, d))
    _check(v_pages, "v_pages", dev, q.dtype, (pages, kv_heads, page_size, d))
    _check(table, "table", dev, torch.int32, (slots, table.shape[1]))
    _check_ints(lens, "lens", dev, (slots,))
    if out is None:
        out = torch.empty((slots, q_heads, d), dtype=q.dtype, device=dev)
    else:
        _check(out, "out", dev, q.dtype, (slots, q_heads, d))
    for t, what in ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages"), (out, "out"), (table, "table")):
        _inner(t, what)
    lse = torch.empty((slots, q_heads), dtype=torch.float32, device=dev) if return_lse else None
    strides = (ctypes.c_int64 * 11)(*q.stride()[:2], *k_pages.stride()[:3], *v_pages.stride()[:3], *out.stride()[:2],
                                    table.stride(0))
    _call("lc_paged_decode", dev, dtype, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(),
          lse.data_ptr() if return_lse else None, table.data_ptr(), lens.data_ptr(), slots, table.shape[1], pages, page_size,
          q_heads, kv_heads, d, strides, window, sinks, _scale(scale, d), _stream(stream, dev))
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------- pages

def _maps(maps: CacheMaps, what: str = "maps") -> tuple:
    """(device, slots, width, pages) of checked maps."""
    if maps.table.dim() != 2 or maps.refs.dim() != 1:
        raise ValueError(f"{what}: table and refs have 2 and 1 axes")
    dev, (slots, width), pages = maps.table.device, maps.table.shape, maps.refs.shape[0]
    if not maps.table.is_cuda:
        raise ValueError(f"{what}: on {dev}, the kernels run on CUDA devices only")
    _check_ints(maps.table, f"{what}.table", dev, (slots, width))
    _check_ints(maps.lens, f"{what}.lens", dev, (slots,))
    _check_ints(maps.refs, f"{what}.refs", dev, (pages,))
    if maps.status is not None:
        _check_ints(maps.status, f"{what}.status", dev, (2,))
    return dev, slots, width, pages


def _into(maps: CacheMaps, into: CacheMaps | None) -> CacheMaps:
    """The maps an operation writes: new ones, or the given ones with a status."""
    if into is None:
        return CacheMaps(torch.empty_like(maps.table), torch.empty_like(maps.lens), torch.empty_like(maps.refs),
                         torch.empty(2, dtype=torch.int32, device=maps.table.device))
    if _maps(into, "into") != _maps(maps):
        raise ValueError("into: other sizes or another device than the maps")
    return into if into.status is not None else into._replace(status=torch.empty(2, dtype=torch.int32, device=into.table.device))


def _pool(pool, dev, pages: int) -> tuple:
    """The pool's arguments of the page operations: pointer, planes, heads, bytes of a token, strides; and page_size."""
    if pool.dim() != 5 or pool.device != dev or pool.shape[1] != pages:
        raise ValueError(f"pool: {tuple(pool.shape)} on {pool.device}, expected [planes, {pages}, kv_heads, page_size, d] on {dev}")
    planes, _, heads, page_size, d = pool.shape
    _inner(pool, "pool")
    if page_size > 1 and pool.stride(3) != d:
        raise ValueError("pool: the tokens of a head must be contiguous")
    size = pool.element_size()
    strides = (ctypes.c_int64 * 3)(*(s * size for s in pool.stride()[:3]))
    return (pool.data_ptr(), planes, heads, d * size, strides), page_size


def cache_extend(maps: CacheMaps, add, *, page_size: int, into: CacheMaps | None = None, stream: int | None = None) -> CacheMaps:
    """Room for ``add[slots]`` more tokens: pages are taken (the lowest free ones, in slot order) and ``lens`` grow.

    All or nothing: where pages or table columns are missing, the maps stay as they are and ``status`` says so.
    """
    dev, slots, width, pages = _maps(maps)
    _check_ints(add, "add", dev, (slots,))
    new = _into(maps, into)
    _call("lc_cache_extend", dev, maps.table.data_ptr(), new.table.data_ptr(), maps.lens.data_ptr(), new.lens.data_ptr(),
          maps.refs.data_ptr(), new.refs.data_ptr(), add.data_ptr(), new.status.data_ptr(), slots, width, pages, page_size,
          _stream(stream, dev))
    return new


def cache_write(k, v, k_pages, v_pages, maps: CacheMaps, add, *, stream: int | None = None) -> None:
    """Writes the newest ``add[i]`` tokens of every slot, ``k, v[slots, most, kv_heads, d]``, to the positions
    ``lens[i] - add[i]`` and on (``maps`` as :func:`cache_extend` left them).  ``k_pages, v_pages[pages, kv_heads,
    page_size, d]`` are planes of the pool; any element type."""
    dev, slots, width, pages = _maps(maps)
    _check_ints(add, "add", dev, (slots,))
    if k.dim() != 4 or k_pages.dim() != 4:
        raise ValueError(f"k and k_pages have 4 axes, got {k.dim()} and {k_pages.dim()}")
    _, most, heads, d = k.shape
    page_size, size = k_pages.shape[2], k.element_size()
    for t, what in ((k, "k"), (v, "v")):
        _check(t, what, dev, k.dtype, (slots, most, heads, d))
        _inner(t, what)
    for t, what in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        _check(t, what, dev, k.dtype, (pages, heads, page_size, d))
        _inner(t, what)
    strides = (ctypes.c_int64 * 12)(*(s * size for t in (k, v, k_pages, v_pages) for s in t.stride()[:3]))
    _call("lc_cache_write", dev, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), maps.table.data_ptr(),
          maps.lens.data_ptr(), add.data_ptr(), slots, most, width, pages, page_size, heads, d * size, strides,
          _stream(stream, dev))


def cache_fork(pool, maps: CacheMaps, parent, *, into: CacheMaps | None = None, stream: int | None = None) -> CacheMaps:
    """Slot ``i`` goes on as slot ``parent[i]`` was (-1: it is dropped): samples of one prompt, or beams that reorder.

    Full pages are shared.  A last page that is not full stays with the lowest slot of its parent; the others get a
    page of their own (the lowest free ones, in slot order) with its tokens.  All or nothing, as :func:`cache_extend`;
    the new maps may not be the old ones.
    """
    dev, slots, width, pages = _maps(maps)
    _check_ints(parent, "parent", dev, (slots,))
    args, page_size = _pool(pool, dev, pages)
    new = _into(maps, into)
    _call("lc_cache_fork", dev, *args, maps.table.data_ptr(), new.table.data_ptr(), maps.lens.data_ptr(), new.lens.data_ptr(),
          maps.refs.data_ptr(), new.refs.data_ptr(), parent.data_ptr(), new.status.data_ptr(), slots, width, pages, page_size,
          _stream(stream, dev))
    return new


def _release(maps, gone, window, sinks, page_size, stream) -> CacheMaps:
    dev, slots, width, pages = _maps(maps)
    if gone is not None:
        _check_ints(gone, "gone", dev, (slots,))
    maps = _into(maps, maps)
    _call("lc_cache_release", dev, maps.table.data_ptr(), maps.lens.data_ptr(), maps.refs.data_ptr(),
          gone.data_ptr() if gone is not None else None, window, sinks, maps.status.data_ptr(), slots, width, pages, page_size,
          _stream(stream, dev))
    return maps


def cache_release(maps: CacheMaps, gone, *, page_size: int, stream: int | None = None) -> CacheMaps:
    """Empties the slots with ``gone[i] != 0`` and gives their pages back, in place."""
    return _release(maps, gone, 0, 0, page_size, stream)


def cache_trim(maps: CacheMaps, *, window: int, sinks: int = 0, page_size: int, stream: int | None = None) -> CacheMaps:
    """Gives back, in place, the pages that no token to come will see under this window and these sinks."""
    return _release(maps, None, window, sinks, page_size, stream)


def cache_compact(pool, maps: CacheMaps, *, into: CacheMaps | None = None, stream: int | None = None) -> CacheMaps:
    """Moves the pages in use onto the lowest numbers (``pages - status[1]`` of them); tables and refs follow."""
    dev, slots, width, pages = _maps(maps)
    args, page_size = _pool(pool, dev, pages)
    new = _into(maps, into)
    _call("lc_cache_compact", dev, *args, maps.table.data_ptr(), new.table.data_ptr(), maps.lens.data_ptr(),
          new.lens.data_ptr(), maps.refs.data_ptr(), new.refs.data_ptr(), new.status.data_ptr(), slots, width, pages, page_size,
          _stream(stream, dev))
    return new


def cache_copy(pool, src, dst, *, stream: int | None = None) -> None:
    """Copies page ``src[i]`` onto page ``dst[i]`` in every plane (int32 on the device).  No page may be a destination
    twice, or a destination and a source."""
    dev, pages = pool.device, pool.shape[1]
    if not pool.is_cuda:
        raise ValueError(f"pool: on {dev}, the kernels run on CUDA devices only")
    _check_ints(src, "src", dev, (src.numel(),))
    _check_ints(dst, "dst", dev, (src.numel(),))
    args, page_size = _pool(pool, dev, pages)
    _call("lc_cache_copy", dev, *args, src.data_ptr(), dst.data_ptr(), src.numel(), pages, page_size, _stream(stream, dev))


class PagedCache:
    """The keys and values of ``layers`` attention layers of up to ``slots`` sequences, in pages.

    ``pool[2 * layers, pages, kv_heads, page_size, head_dim]`` holds layer ``l``'s keys in plane ``2 l`` and its values
    in plane ``2 l + 1``; ``maps`` are its :class:`CacheMaps`.  Every method works on the device, in stream order;
    :meth:`check` waits for it and raises where an operation could not be done.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int, width: int,
                 dtype=torch.bfloat16, device="cuda"):
        if min(layers, pages, page_size, kv_heads, head_dim, slots, width) < 1:
            raise ValueError("every size of a PagedCache is at least 1")
        self.pool = torch.zeros((2 * layers, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=self.pool.device)
        self.page_size = page_size
        self.maps, self._spare = (CacheMaps(torch.full((slots, width), -1, **ints), torch.zeros(slots, **ints),
                                            torch.zeros(pages, **ints), torch.zeros(2, **ints)) for _ in range(2))
        self.maps.status[1] = pages

    def extend(self, add, stream=None) -> None:
        """Room for ``add[slots]`` more tokens (:func:`cache_extend`)."""
        cache_extend(self.maps, add, page_size=self.page_size, into=self.maps, stream=stream)

    def write(self, layer: int, k, v, add, stream=None) -> None:
        """The newest tokens' keys and values of one layer (:func:`cache_write`)."""
        cache_write(k, v, self.pool[2 * layer], self.pool[2 * layer + 1], self.maps, add, stream=stream)

    def decode(self, layer: int, q, **options):
        """Attention of one new token per slot in one layer (:func:`paged_decode`)."""
        return paged_decode(q, self.pool[2 * layer], self.pool[2 * layer + 1], self.maps.table, self.maps.lens, **options)

    def fork(self, parent, stream=None) -> None:
        """Slots continue others (:func:`cache_fork`).  The maps are other tensors afterwards."""
        cache_fork(self.pool, self.maps, parent, into=self._spare, stream=stream)
        self.maps, self._spare = self._spare, self.maps

    def release(self, gone, stream=None) -> None:
        """Empties slots (:func:`cache_release`)."""
        cache_release(self.maps, gone, page_size=self.page_size, stream=stream)

    def trim(self, window: int, sinks: int = 0, stream=None) -> None:
        """Gives back what a sliding window has left behind (:func:`cache_trim`)."""
        cache_trim(self.maps, window=window, sinks=sinks, page_size=self.page_size, stream=stream)

    def compact(self, stream=None) -> None:
        """Moves the pages in use onto the lowest numbers (:func:`cache_compact`)."""
        cache_compact(self.pool, self.maps, into=self.maps, stream=stream)

    def check(self) -> int:
        """Waits for the last operation on the maps; the pages free after it, or an error where it was refused."""
        code, free = self.maps.status.tolist()
        if code:
            what = "an argument is out of range" if code < 0 else f"{code} pages are missing"
            raise RuntimeError(f"the cache is unchanged: {what} ({free} pages are free)")
        return free
