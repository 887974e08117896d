"""Serving operators: attention of prompts and of single new tokens, the paged key-value cache between them, and what a
step has around them: positions as rotations, and the drawing of the next token.

The functions take torch tensors on one CUDA device and launch the library's kernels (``include/lazyb200.h``,
"serving") on the tensors' device, on its current stream or on ``stream``:

* :func:`window_attention` — a prompt, or the next chunk of one, over its keys: causal, optionally with a sliding
  window and a few first tokens ("sinks") that stay visible;
* :func:`paged_decode` — one new token per sequence over the pages of its keys and values;
* :func:`shared_decode` — the same where sequences begin with the same pages: samples of a prompt, questions to a
  document.  What they share, as :func:`cache_prefixes` finds it, is read once;
* :func:`rotate` — positions as rotations of queries and keys, by a :class:`Rotary`'s frequencies;
* :func:`cache_append` — a layer's new tokens on their way: queries and keys turned, keys and values into their pages;
* :func:`sample` — a token of every row of logits, by temperature, top-k, top-p and min-p, from given uniform numbers;
* :func:`cache_extend`, :func:`cache_write`, :func:`cache_fork`, :func:`cache_release`, :func:`cache_trim`,
  :func:`cache_compact`, :func:`cache_copy` — the pages themselves.

A cache is a ``pool[planes, pages, kv_heads, page_size, head_dim]`` (a plane is the keys or the values of one layer)
and its :class:`CacheMaps`, int32 tensors on the device.  What is free is read from ``refs`` alone, so no operation
needs the host: a decode step can be captured in a CUDA graph.  Operations on maps return new ones, or write ``into``
given ones, which may be the same (not for :func:`cache_fork`).  :class:`PagedCache` keeps a pool with its maps.

A tensor used on another stream than the one it was made on needs ``record_stream`` or an event, as any torch tensor;
what a call with ``stream`` returns was made on that one.
The waits inside the kernels of the prompt form and of shared prefixes are bounded.  One that runs out (a fault of the machine) leaves outputs
unwritten; ``runtime.call("lc_device_status", stream)`` tells of it, as :meth:`PagedCache.check` does.

No operation has a gradient: with grad mode on, an input that requires one is refused.

The library's workspaces belong to a stream and grow on its first calls: before a capture, run the step once on the
stream that will capture it.  A graph keeps the workspaces of the stream it was captured on, also when later calls make
them grow; so graphs captured on one stream, and calls on that stream, may not run at the same time.
"""
from __future__ import annotations

import ctypes
import math
from fractions import Fraction
from typing import NamedTuple

import torch

from . import runtime

# the order in which csrc/serving_ext.cpp takes the entry points
_ENTRIES = ("lc_window_attention", "lc_paged_decode", "lc_cache_extend_recorded", "lc_cache_write_unless",
            "lc_cache_fork_recorded", "lc_cache_release", "lc_cache_compact", "lc_cache_copy")
_STEP_ENTRIES = ("lc_rotate", "lc_cache_append", "lc_cache_prefixes", "lc_sample", "lc_shared_decode")


def _extension():
    """The extension module, bound to the loaded library.  There is no other path: unbuilt, this raises."""
    library = runtime.library()
    try:
        from . import _serving
    except ImportError as e:
        raise RuntimeError("the extension module _serving is not built; run `python -m lazy_compiler_b200.build`") from e
    for bind, names in ((_serving.bind, _ENTRIES), (_serving.bind_steps, _STEP_ENTRIES)):
        bind(*(ctypes.cast(getattr(library, name), ctypes.c_void_p).value for name in names))
    return _serving


_ext = _extension()


def _failed(name: str, status: int):
    """The error of a C-ABI call."""
    return runtime.LcError(name, status, runtime.last_error())


class CacheMaps(NamedTuple):
    """Whose pages are whose: ``table[slots, width]`` (a sequence's pages in order, -1 where there is none),
    ``lens[slots]`` (its tokens), ``refs[pages]`` (how many sequences hold the page) and, from the operation that
    made them, ``status[2]``: 0, -1 (an argument out of range) or the number of pages missing, where it is not 0 the
    maps are unchanged; and the pages free."""
    table: torch.Tensor
    lens: torch.Tensor
    refs: torch.Tensor
    status: torch.Tensor | None = None


def window_attention(q, k, v, *, window: int = 0, sinks: int = 0, scale: float | None = None, q_lens=None, kv_lens=None,
                     out=None, return_lse: bool = False, stream: int | None = None):
    """Causal attention of ``q[batch, s_q, q_heads, d]`` over ``k, v[batch, s_kv, kv_heads, d]`` (f16 or bf16).

    Sequence ``b`` has ``q_lens[b]`` queries and ``kv_lens[b]`` keys (int32 on the device; all of them by default);
    its query ``i`` is at position ``p = kv_lens[b] - q_lens[b] + i`` and sees key ``j <= p`` when ``window`` is 0,
    ``j > p - window`` or ``j < sinks``.  ``scale`` is ``1 / sqrt(d)`` by default.  Returns ``o`` like ``q`` (``out``
    where given), with ``return_lse`` also the log-sum-exp of the scaled scores, f32 ``[batch, q_heads, s_q]``.  Rows
    that see nothing, and rows from ``q_lens[b]`` on, are 0 and -inf.  Any strides with a contiguous last axis; ``out``
    overlaps no input.
    """
    r = _ext.window_attention(q, k, v, window, sinks, scale, q_lens, kv_lens, out, return_lse, stream)
    if type(r) is int:
        raise _failed("lc_window_attention", r)
    return r


def paged_decode(q, k_pages, v_pages, table, lens, *, window: int = 0, sinks: int = 0, scale: float | None = None, out=None,
                 return_lse: bool = False, stream: int | None = None):
    """Attention of one new token per sequence, ``q[slots, q_heads, d]``, over its cached keys and values.

    ``k_pages, v_pages[pages, kv_heads, page_size, d]`` (a pool's planes), ``table[slots, width]`` and ``lens[slots]``
    as in :class:`CacheMaps`; ``lens`` counts the new token, whose key and value are in the cache already.  The rest
    is as in :func:`window_attention`, of which this is the single-token form; the log-sum-exp is ``[slots, q_heads]``.
    """
    r = _ext.paged_decode(q, k_pages, v_pages, table, lens, window, sinks, scale, out, return_lse, stream)
    if type(r) is int:
        raise _failed("lc_paged_decode", r)
    return r


# ---------------------------------------------------------------- positions

class Rotary:
    """How positions enter queries and keys: the first ``dim`` elements of a head are pairs, ``(i, i + dim / 2)`` or
    ``interleaved`` ``(2 i, 2 i + 1)``, and pair ``i`` at position ``p`` turns by the angle ``p f[i]``.

    ``f[i]`` is ``base ** (-2 i / dim)``, for contexts longer than trained by ``factor`` with one of the ``scaling``:

    * ``"linear"`` — ``f / factor``, every position interpolated;
    * ``"base"`` — ``base * factor ** (dim / (dim - 2))``: the slowest pair is interpolated, the fastest stays;
    * ``"bands"`` — pairs that turn ``fast`` times or more over the ``trained`` context stay, those that turn ``slow``
      times or fewer are interpolated, a linear ramp in the turns between them; and the turned elements are multiplied
      by ``magnitude``, here ``1 + 0.1 ln factor`` by default (1 elsewhere);

    or ``frequencies`` (radians a position, float64 ``[dim / 2]``) are given.  ``turns[dim / 2]``, int64 on the device,
    holds them as fractions of a turn, in units of 2^-64: angles are exact at any position.
    """

    def __init__(self, dim: int, base: float = 10000.0, *, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
                 trained: int = 0, slow: float = 1.0, fast: float = 32.0, magnitude: float | None = None, frequencies=None, device="cuda"):
        if dim < 0 or dim % 2:
            raise ValueError(f"dim: {dim} elements are not pairs")
        if scaling not in ("none", "linear", "base", "bands"):
            raise ValueError(f"scaling: {scaling!r} is not none, linear, base or bands")
        if not 0 < base < math.inf or not 0 < factor < math.inf:
            raise ValueError("base and factor are positive")
        if scaling == "none" and factor != 1.0:
            raise ValueError("factor: there is no scaling")
        if scaling == "base" and dim <= 2:
            raise ValueError("scaling: a single pair turns by one radian whatever the base")
        if scaling == "bands" and not (trained > 0 and 0 <= slow < fast):
            raise ValueError("scaling: bands need the trained context, and slow < fast")
        if frequencies is not None:
            f = torch.as_tensor(frequencies, dtype=torch.float64).cpu()
            if scaling != "none" or f.shape != (dim // 2,):
                raise ValueError(f"frequencies: shape {tuple(f.shape)}, expected ({dim // 2},), and no scaling beside them")
        else:
            stretched = base * factor ** (dim / (dim - 2)) if scaling == "base" else base
            f = stretched ** (-torch.arange(0, dim, 2, dtype=torch.float64) / max(1, dim))
        if scaling == "linear":
            f = f / factor
        if scaling == "bands":
            stays = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
            f = f * (stays + (1 - stays) / factor)
        if not bool((f.abs() < 2.0 ** 31).all()):
            raise ValueError("frequencies: not finite, or a position turns by more than 2^31 radians")
        self.dim, self.interleaved, self.frequencies = dim, bool(interleaved), f
        self.magnitude = float(magnitude) if magnitude is not None else 1 + 0.1 * math.log(factor) if scaling == "bands" else 1.0
        if not 0 < self.magnitude < 3e38:
            raise ValueError("magnitude: must be positive and finite")
        # whole turns change nothing; the fraction to 64 bits, half a turn and more as its negative
        turns = [_turns(x) % 2 ** 64 for x in f.tolist()]
        self.turns = torch.tensor([t - 2 ** 64 if t >> 63 else t for t in turns], dtype=torch.int64).to(device)


# a turn in radians, to 130 bits or so: pi by Machin's formula
def _arctan_inverse(n: int) -> Fraction:
    return sum(Fraction((-1) ** k, (2 * k + 1) * n ** (2 * k + 1)) for k in range(30))


_TURN = 8 * (4 * _arctan_inverse(5) - _arctan_inverse(239))
_TURNS = round(2 ** 192 / _TURN)  # of a radian, in units of 2^-192


def _turns(radians: float) -> int:
    """Of an angle, in units of 2^-64."""
    top, bottom = radians.as_integer_ratio()  # bottom is a power of two
    return (2 * top * _TURNS // (bottom << 128) + 1) // 2


def rotate(x, positions, rotary: Rotary, *, out=None, stream: int | None = None):
    """``x[batch, tokens, heads, d]`` (f32, f16 or bf16; any strides with a contiguous last axis) with every head turned to
    its token's place, ``positions[batch, tokens]`` (int32 on the device; negative ones turn back).

    Elements behind ``rotary.dim`` pass.  The arithmetic is f32, rounded once.  ``out`` may be ``x`` itself, and overlaps
    it in no other way.
    """
    r = _ext.rotate(x, positions, rotary.turns, rotary.interleaved, rotary.magnitude, out, stream)
    if type(r) is int:
        raise _failed("lc_rotate", r)
    return r


# ---------------------------------------------------------------- tokens

def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, return_logprob: bool = False,
           stream: int | None = None):
    """A token of each row of ``logits[rows, vocab]`` (f32, f16 or bf16; any stride between rows), int32 ``[rows]``.

    With the weights ``w = exp((x - max) / temperature)``, what is kept is the ``top_k`` largest, of these the shortest run
    from the largest on that holds ``top_p`` of their sum, of these those with ``w >= min_p``; the token is the first index
    at which the running sum of what is kept passes ``uniform[row]`` (f32, in [0, 1)) times its total.  Equal logits are
    taken in index order.  ``temperature`` 0 takes the largest; ``top_k`` 0 (or ``vocab`` and more), ``top_p`` 1 and
    ``min_p`` 0 leave all.  Each is a number, or a tensor of one a row (f32, ``top_k`` int32).  NaN and -infinity are never
    taken: a row of nothing else gives -1.

    With ``return_logprob`` also the logarithm of the token's share of what was kept, f32 ``[rows]``.  Sums are exact (whole
    numbers), so a row's token depends on nothing but the row.
    """
    r = _ext.sample(logits, uniform, temperature, top_k, top_p, min_p, out, return_logprob, stream)
    if type(r) is int:
        raise _failed("lc_sample", r)
    return r


# ---------------------------------------------------------------- pages

_NONE = (None, None, None, None)


def cache_extend(maps: CacheMaps, add, *, page_size: int, into: CacheMaps | None = None, refusals=None,
                 stream: int | None = None) -> CacheMaps:
    """Room for ``add[slots]`` more tokens: pages are taken (the lowest free ones, in slot order) and ``lens`` grow.

    All or nothing: where pages or table columns are missing, the maps stay as they are and ``status`` says so.  The
    next operation writes another status; ``refusals[2]`` (int32 on the device) keeps the first one that was not 0 in
    ``refusals[0]`` until the caller clears it, and that of the last extension in ``refusals[1]``.
    """
    r = _ext.cache_extend(*maps, add, page_size, *(into or _NONE), refusals, stream)
    if type(r) is int:
        raise _failed("lc_cache_extend", r)
    return CacheMaps(*r)


def cache_write(k, v, k_pages, v_pages, maps: CacheMaps, add, *, refusals=None, stream: int | None = None) -> None:
    """Writes the newest ``add[i]`` tokens of every slot, ``k, v[slots, most, kv_heads, d]``, to the positions
    ``lens[i] - add[i]`` and on (``maps`` as :func:`cache_extend` left them).  ``k_pages, v_pages[pages, kv_heads,
    page_size, d]`` are planes of the pool; any element type.  Where ``refusals[1]``, or without them ``maps.status[0]``, is
    not 0 (room was refused, and ``lens`` did not grow) nothing is written: the positions are those of tokens that are
    there."""
    status = _ext.cache_write(k, v, k_pages, v_pages, *maps, add, refusals, stream)
    if status:
        raise _failed("lc_cache_write", status)


def cache_append(q, k, v, k_pages, v_pages, maps: CacheMaps, add, rotary: Rotary, *, out=None, refusals=None,
                 stream: int | None = None):
    """:func:`cache_write` with the positions on the way: the newest ``add[i]`` tokens' keys, turned to the positions
    ``lens[i] - add[i]`` and on (:func:`rotate`), and values go to their pages, and ``q[slots, most, q_heads, d]`` comes back
    turned alike (``None`` where ``q`` is).

    f32, f16 or bf16, the pages of the same type.  Queries behind ``add[i]`` come back as 0; in a given ``out``, which may
    be ``q`` itself, they are left as they were.  After a refused extension (as in :func:`cache_write`) no token is new.
    """
    r = _ext.cache_append(q, k, v, k_pages, v_pages, *maps, add, rotary.turns, rotary.interleaved, rotary.magnitude, out, refusals, stream)
    if type(r) is int:
        raise _failed("lc_cache_append", r)
    return r


def cache_fork(pool, maps: CacheMaps, parent, *, into: CacheMaps | None = None, refusals=None, stream: int | None = None) -> CacheMaps:
    """Slot ``i`` goes on as slot ``parent[i]`` was (-1: it is dropped): samples of one prompt, or beams that reorder.

    Full pages are shared.  A last page that is not full stays with the lowest slot of its parent; the others get a
    page of their own (the lowest free ones, in slot order) with its tokens.  All or nothing, as :func:`cache_extend`;
    the new maps may not be the old ones.  ``refusals[0]`` is kept as there.
    """
    r = _ext.cache_fork(pool, *maps, parent, *(into or _NONE), refusals, stream)
    if type(r) is int:
        raise _failed("lc_cache_fork", r)
    return CacheMaps(*r)


def _release(maps, gone, window, sinks, page_size, stream) -> CacheMaps:
    r = _ext.cache_release(*maps, gone, window, sinks, page_size, stream)
    if type(r) is int:
        raise _failed("lc_cache_release", r)
    return CacheMaps(*r)


def cache_release(maps: CacheMaps, gone, *, page_size: int, stream: int | None = None) -> CacheMaps:
    """Empties the slots with ``gone[i] != 0`` and gives their pages back, in place."""
    return _release(maps, gone, 0, 0, page_size, stream)


def cache_trim(maps: CacheMaps, *, window: int, sinks: int = 0, page_size: int, stream: int | None = None) -> CacheMaps:
    """Gives back, in place, the pages that no token to come will see under this window and these sinks."""
    return _release(maps, None, window, sinks, page_size, stream)


def cache_compact(pool, maps: CacheMaps, *, into: CacheMaps | None = None, stream: int | None = None) -> CacheMaps:
    """Moves the pages in use onto the lowest numbers (``pages - status[1]`` of them); tables and refs follow."""
    r = _ext.cache_compact(pool, *maps, *(into or _NONE), stream)
    if type(r) is int:
        raise _failed("lc_cache_compact", r)
    return CacheMaps(*r)


def cache_copy(pool, src, dst, *, stream: int | None = None) -> None:
    """Copies page ``src[i]`` onto page ``dst[i]`` in every plane (int32 on the device).  No page may be a destination
    twice, or a destination and a source."""
    status = _ext.cache_copy(pool, src, dst, stream)
    if status:
        raise _failed("lc_cache_copy", status)


class CachePrefixes(NamedTuple):
    """Which slots begin with the same pages: ``leader[slots]`` (the lowest slot with the same full first page),
    ``shared[slots]`` (the tokens of the full pages that all slots of that leader have in common; 0 for a slot alone) and
    ``order[slots]`` (the slots by leader, each group in slot order)."""
    leader: torch.Tensor
    shared: torch.Tensor
    order: torch.Tensor


def cache_prefixes(maps: CacheMaps, *, page_size: int, into: CachePrefixes | None = None, stream: int | None = None) -> CachePrefixes:
    """Which slots begin with the same pages, and how far: what :func:`cache_fork` leaves of one prompt.  At most 8192
    slots.  It holds until a slot is forked, released or trimmed: what is extended, written or compacted keeps its
    prefix."""
    r = _ext.cache_prefixes(*maps, page_size, *(into or (None, None, None)), stream)
    if type(r) is int:
        raise _failed("lc_cache_prefixes", r)
    return CachePrefixes(*r)


def shared_decode(q, k_pages, v_pages, table, lens, prefixes: CachePrefixes, *, window: int = 0, sinks: int = 0,
                  scale: float | None = None, out=None, return_lse: bool = False, stream: int | None = None):
    """:func:`paged_decode` for slots that begin alike: samples of one prompt, questions to one document.

    ``prefixes`` is what :func:`cache_prefixes` found, or the same in other tensors: slots with one leader lie together in
    ``order``, the leader first, and hold its pages over the first ``shared[leader]`` tokens.  Such a prefix is read once
    for all of them.  At most 8192 slots; the rest is as there.
    """
    r = _ext.shared_decode(q, k_pages, v_pages, table, lens, *prefixes, window, sinks, scale, out, return_lse, stream)
    if type(r) is int:
        raise _failed("lc_shared_decode", r)
    return r


class PagedCache:
    """The keys and values of ``layers`` attention layers of up to ``slots`` sequences, in pages.

    ``pool[2 * layers, pages, kv_heads, page_size, head_dim]`` holds layer ``l``'s keys in plane ``2 l`` and its values
    in plane ``2 l + 1``; ``maps`` are its :class:`CacheMaps`, the same tensors always.  Every method works on the
    device, in stream order; :meth:`check` waits for it and raises where one could not be done since the check before.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int, width: int,
                 dtype=torch.bfloat16, device="cuda"):
        if min(layers, pages, page_size, kv_heads, head_dim, slots, width) < 1:
            raise ValueError("every size of a PagedCache is at least 1")
        self.pool = torch.zeros((2 * layers, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=self.pool.device)
        self.page_size = page_size
        # the maps, and those that a fork writes; each set is one block of memory
        self._blocks = [torch.zeros(slots * width + slots + pages + 2, **ints) for _ in range(2)]
        self._own, self._spare = (CacheMaps(t.view(slots, width), n, r, s) for t, n, r, s in
                                  (b.split([slots * width, slots, pages, 2]) for b in self._blocks))
        self.maps = self._own
        self.maps.table.fill_(-1)
        self.maps.status[1] = pages
        self._refusals = torch.zeros(2, **ints)

    def extend(self, add, stream=None) -> None:
        """Room for ``add[slots]`` more tokens (:func:`cache_extend`)."""
        cache_extend(self.maps, add, page_size=self.page_size, into=self.maps, refusals=self._refusals, stream=stream)

    def write(self, layer: int, k, v, add, stream=None) -> None:
        """The newest tokens' keys and values of one layer (:func:`cache_write`); nothing where the last
        :meth:`extend` was refused."""
        cache_write(k, v, self.pool[2 * layer], self.pool[2 * layer + 1], self.maps, add, refusals=self._refusals, stream=stream)

    def append(self, layer: int, q, k, v, add, rotary: Rotary, out=None, stream=None):
        """The same with the keys turned to their positions; returns the queries turned to theirs (:func:`cache_append`)."""
        return cache_append(q, k, v, self.pool[2 * layer], self.pool[2 * layer + 1], self.maps, add, rotary, out=out,
                            refusals=self._refusals, stream=stream)

    def decode(self, layer: int, q, **options):
        """Attention of one new token per slot in one layer (:func:`paged_decode`)."""
        return paged_decode(q, self.pool[2 * layer], self.pool[2 * layer + 1], self.maps.table, self.maps.lens, **options)

    def shared_decode(self, layer: int, q, prefixes: CachePrefixes, **options):
        """The same where slots begin alike (:func:`shared_decode`)."""
        return shared_decode(q, self.pool[2 * layer], self.pool[2 * layer + 1], self.maps.table, self.maps.lens, prefixes, **options)

    def fork(self, parent, stream=None) -> None:
        """Slots continue others (:func:`cache_fork`).  The new maps are copied back into the same tensors, so that a
        step captured before goes on with them."""
        cache_fork(self.pool, self.maps, parent, into=self._spare, refusals=self._refusals, stream=stream)
        with torch.cuda.stream(None if stream is None else torch.cuda.ExternalStream(stream, self.pool.device)):
            self._blocks[0].copy_(self._blocks[1])
        self.maps = self._own  # where the caller had put others in their place

    def prefixes(self, into: CachePrefixes | None = None, stream=None) -> CachePrefixes:
        """Which slots begin with the same pages (:func:`cache_prefixes`)."""
        return cache_prefixes(self.maps, page_size=self.page_size, into=into, stream=stream)

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
        """Waits for the last operation on the maps (on the current stream, or one that it waits for); the pages free
        after it.  Raises where an operation could not be done, the first of them since the last check, whatever came
        after it, and where a kernel gave up a wait inside it (``lc_device_status``)."""
        code, free, refused, _ = torch.cat((self.maps.status, self._refusals)).tolist()
        code = refused or code
        if code:
            self._refusals[0] = 0
            what = "an argument is out of range" if code < 0 else f"{code} pages are missing"
            raise RuntimeError(f"an operation was refused and changed nothing: {what} ({free} pages are free)")
        with torch.cuda.device(self.pool.device):
            runtime.call("lc_device_status", torch.cuda.current_stream().cuda_stream)
        return free
