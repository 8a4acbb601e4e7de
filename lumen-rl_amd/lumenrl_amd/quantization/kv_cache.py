"""The FP8 KV cache: paged keys and values in e4m3, attention over them, and their pages' upkeep.

``FP8KVCache`` holds a model's pages.  Sequences are rows of a page table that the
caller keeps: ``table`` int32 [rows, width] with a row's page numbers in order and
``lengths`` int32 [rows].  A step of a rollout is

    table, lengths, short, ready = cache.resize(table, lengths, lengths + new, return_ready=True)   # once
    cache.append(layer, k, v, table, ready, offsets)                                                # in each layer
    out = cache.attend(layer, q, table, ready, offsets)

``ready`` is 0 for a row that there was no room for: its new tokens are written nowhere, see
nothing and get 0, and ``lengths`` still says what it has.  (With ``lengths`` in its place
the row's last tokens would be taken for the new ones, and overwritten.)  ``fork`` makes
samples of a prompt share its pages, ``resize`` to 0 ends a sequence, ``compact`` moves what
is left together.  Everything runs on the current stream of the
cache's device, reads lengths and tables there, and returns without synchronizing, so a
step can be captured into a graph.  Calls that write a page are the caller's to keep in order
with others on that page, ``fork``, ``resize`` and ``compact`` with each other.  What tables,
lengths and offsets hold is clamped to what there is: an entry that is no page of the pool is
no page.  Offsets do not go back; what becomes of rows that two sequences claim is open.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
from torch import Tensor, UntypedStorage
from torch.autograd import forward_ad

from lumenrl_amd import _lib
from lumenrl_amd.quantization.fp8_product import NoGradient
from lumenrl_amd.quantization.ops import _IN_DTYPES, _check_input, _current_device, _dense, _on, _stream, require_device

_STRIDE_MAX = 1 << 40
_WINDOW_MAX = 1 << 31  # more than a sequence can have
_SCALE_MAX = 2.0 ** 127  # that of float32, in base 2, has an exponent of one more


@functools.lru_cache(maxsize=4096)
def _append_workspace(seqs: int) -> int:
    return _lib.lib().lrq_kv_append_workspace(seqs, False)


@functools.lru_cache(maxsize=4096)
def _attend_workspace(tokens: int, heads: int, kv_heads: int, dim: int, seqs: int, one_each: bool) -> int:
    return _lib.lib().lrq_kv_attend_workspace(tokens, heads, kv_heads, dim, seqs, one_each)


@functools.lru_cache(maxsize=4096)
def _resize_workspace(rows: int, pages: int) -> int:
    return _lib.lib().lrq_kv_resize_workspace(rows, pages)


@functools.lru_cache(maxsize=4096)
def _compact_workspace(pages: int) -> int:
    return _lib.lib().lrq_kv_compact_workspace(pages)


def _steps(name: str, x: Tensor, inner: int) -> tuple[int, int]:
    """Strides from layer to layer and page to page of a tensor whose other ``inner`` dims are dense."""
    if x.numel() == 0:
        return 0, 0
    step = 1
    for d in range(x.dim() - 1, x.dim() - 1 - inner, -1):
        if x.shape[d] > 1 and x.stride(d) != step:
            raise ValueError(f"FP8KVCache: a page of {name} must be dense, got strides {x.stride()}")
        step *= x.shape[d]
    if x.shape[1] > 1 and x.stride(1) < step:
        raise ValueError(f"FP8KVCache: pages of {name} overlap (strides {x.stride()})")
    return x.stride(0), x.stride(1)


def _places(parts: tuple) -> list:
    """Where tensors are, and how long the memory is that they are in."""
    return [*map(Tensor.data_ptr, parts), *map(UntypedStorage.nbytes, map(Tensor.untyped_storage, parts))]


def _part(i: int) -> property:
    """One of a cache's tensors: to be written to (``cache.refs += 1`` too), not to be replaced."""

    def keep(self, x: Tensor) -> None:
        if x is not self._parts[i]:
            raise AttributeError("FP8KVCache: its tensors cannot be replaced; make another cache of the new ones")

    return property(lambda self: self._parts[i], keep)


def _wants_derivative(x: Tensor, y: Tensor) -> bool:
    """Whether one of them is to be differentiated, backward or forward."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, y)):
        return True
    return (x.requires_grad or y.requires_grad) and torch.is_grad_enabled()


class FP8KVCache:
    """Pages of keys and values in e4m3, with one power-of-two scale per page and KV head for each.

    ``k`` [layers, pages, kv_heads, page, dim] and ``v`` [layers, pages, kv_heads, dim,
    page] are float8_e4m3fn codes, ``k_scales`` and ``v_scales`` [layers, pages,
    kv_heads] float32, ``refs`` [pages] int32: how many rows of the caller's table hold
    each page; it is free where none does.  ``page`` is 16, 32, 64, 128 or 256, ``dim`` a multiple
    of 16 up to 256.  The tensors are kept and written in place; layers and pages may be
    views of larger ones, what a page holds is dense.

    A caller's own scales may be any finite numbers that are not negative; ``attend`` takes V's
    within 2^-48 to 2^48, which ``append`` does not leave, and others as the nearest of these.

    The tensors' memory may be freed and put back between calls (``untyped_storage().resize_``,
    ``.data =``), shapes and strides staying as they are: each call looks where the tensors
    are, and raises where one has no memory, or too little; a captured graph keeps the
    places of its capture.
    """

    def __init__(self, k: Tensor, v: Tensor, k_scales: Tensor, v_scales: Tensor, refs: Tensor) -> None:
        self._parts = (k, v, k_scales, v_scales, refs)
        self._describe()

    k, v, k_scales, v_scales, refs = (_part(i) for i in range(5))

    def _describe(self) -> None:
        """Checks the tensors, and notes where they are for the kernels."""
        k, v, k_scales, v_scales, refs = self._parts
        self._where = None  # until all is well
        parts = {"k": (k, torch.float8_e4m3fn), "v": (v, torch.float8_e4m3fn), "k_scales": (k_scales, torch.float32),
                 "v_scales": (v_scales, torch.float32), "refs": (refs, torch.int32)}
        for name, (x, dtype) in parts.items():
            if not isinstance(x, Tensor) or x.dtype != dtype:
                raise TypeError(f"FP8KVCache: {name} must be a {dtype} tensor, got {x.dtype if isinstance(x, Tensor) else type(x)!r}")
        for name, (x, _) in parts.items():
            if not x.is_cuda or x.device != k.device:
                raise ValueError(f"FP8KVCache: expected {name} on one HIP device, got {x.device}")
        if k.dim() != 5:
            raise ValueError(f"FP8KVCache: k must be [layers, pages, kv_heads, page, dim], got {tuple(k.shape)}")
        self.layers, self.pages, self.kv_heads, self.page, self.dim = k.shape
        if v.shape != (*k.shape[:3], self.dim, self.page):
            raise ValueError(f"FP8KVCache: v must be {(*k.shape[:3], self.dim, self.page)}, got {tuple(v.shape)}")
        if k_scales.shape != k.shape[:3] or v_scales.shape != k.shape[:3]:
            raise ValueError(f"FP8KVCache: scales must be {tuple(k.shape[:3])}, got {tuple(k_scales.shape)} and {tuple(v_scales.shape)}")
        if refs.shape != (self.pages,) or not refs.is_contiguous():
            raise ValueError(f"FP8KVCache: refs must be a contiguous [{self.pages}], got {tuple(refs.shape)}")
        if self.page not in (16, 32, 64, 128, 256) or self.dim % 16 or not 16 <= self.dim <= 256:
            raise ValueError(f"FP8KVCache: pages of {self.page} tokens (16, 32, 64, 128 or 256) and heads of {self.dim} (a multiple of "
                             "16 up to 256)")
        if not 1 <= self.kv_heads <= 256 or not 1 <= self.pages <= 1 << 28 or self.layers > 65536:
            raise ValueError(f"FP8KVCache: {self.layers} layers (at most 65536), {self.pages} pages (1 to 2^28), {self.kv_heads} KV heads "
                             "(1 to 256)")
        for name, (x, _) in parts.items():
            last = x.storage_offset() + sum((n - 1) * step for n, step in zip(x.shape, x.stride()))
            if x.numel() and (last + 1) * x.element_size() > x.untyped_storage().nbytes():
                raise RuntimeError(f"FP8KVCache: the memory of {name} has been freed, or is too small for {tuple(x.shape)}")
        if k.numel() and (k.data_ptr() % 16 or v.data_ptr() % 16):
            raise ValueError("FP8KVCache: k and v must be 16-byte aligned")
        (kl, kp), (vl, vp) = _steps("k", k, 3), _steps("v", v, 3)
        (ksl, ksp), (vsl, vsp) = _steps("k_scales", k_scales, 1), _steps("v_scales", v_scales, 1)
        if any(s % 16 for s in (kl, kp, vl, vp)):
            raise ValueError(f"FP8KVCache: strides of layers and pages must be multiples of 16, got {k.stride()} and {v.stride()}")
        self.device = k.device
        self._index = k.get_device()
        self._desc = _lib.LrqKvCache(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), refs.data_ptr(),
                                     self.layers, self.pages, self.kv_heads, self.page, self.dim, kl, vl, ksl, vsl, kp, vp, ksp, vsp)
        self._ref = ctypes.byref(self._desc)
        self._where = _places(self._parts)

    def _look(self) -> None:
        """First in every call: a caller may have moved the tensors' memory since the last one, or freed it (0.65 us of a call's 7)."""
        if _places(self._parts) != self._where:
            self._describe()

    @classmethod
    def empty(cls, layers: int, pages: int, kv_heads: int, dim: int, *, page: int = 64,
              device: Optional[torch.device] = None) -> "FP8KVCache":
        """A cache with all pages free, on ``device`` (the current one by default)."""
        device = require_device() if device is None else torch.device(device)
        with torch.cuda.device(device):
            k = torch.empty((layers, pages, kv_heads, page, dim), dtype=torch.float8_e4m3fn, device=device)
            v = torch.empty((layers, pages, kv_heads, dim, page), dtype=torch.float8_e4m3fn, device=device)
            ks, vs = (torch.ones((layers, pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2))
            return cls(k, v, ks, vs, torch.zeros(pages, dtype=torch.int32, device=device))

    # -- arguments ---------------------------------------------------------------
    def _ints(self, what: str, name: str, x: Tensor, shape: tuple) -> Tensor:
        if not isinstance(x, Tensor) or x.dtype is not torch.int32:
            raise TypeError(f"{what}: {name} must be an int32 tensor, got {x.dtype if isinstance(x, Tensor) else type(x)!r}")
        if x.shape != shape or x.get_device() != self._index:
            raise ValueError(f"{what}: {name} must be {tuple(shape)} on {self.device}, got {tuple(x.shape)} on {x.device}")
        return x if x.is_contiguous() else x.contiguous()

    def _table(self, what: str, table: Tensor) -> tuple[Tensor, int, int, int]:
        """(table, rows, width, row pitch); a copy only where its rows are not of unit stride."""
        if not isinstance(table, Tensor) or table.dtype is not torch.int32:
            raise TypeError(f"{what}: table must be an int32 tensor, got {table.dtype if isinstance(table, Tensor) else type(table)!r}")
        if table.dim() != 2 or table.get_device() != self._index:
            raise ValueError(f"{what}: table must be [rows, width] on {self.device}, got {tuple(table.shape)} on {table.device}")
        rows, width = table.shape
        if table.is_contiguous():
            return table, rows, width, width
        ld = table.stride(0) if rows > 1 else width
        if (width > 1 and table.stride(1) != 1) or not width <= ld <= _STRIDE_MAX:
            table, ld = table.contiguous(), width
        return table, rows, width, ld

    def _layer(self, what: str, layer: int) -> None:
        if not isinstance(layer, int) or not 0 <= layer < self.layers:
            raise ValueError(f"{what}: layer {layer!r} of {self.layers}")

    def _offsets(self, what: str, offsets: Optional[Tensor], rows: int, tokens: int) -> Optional[Tensor]:
        if offsets is None:
            if tokens < rows:
                raise ValueError(f"{what}: {tokens} tokens of {rows} sequences need offsets")
            return None
        return self._ints(what, "offsets", offsets, (rows + 1,))

    def _vectors(self, what: str, name: str, x: Tensor, heads: Optional[int]) -> Tensor:
        """``x`` [tokens, heads, dim] with channels of unit stride."""
        if not isinstance(x, Tensor) or x.get_device() != self._index or x.dtype not in _IN_DTYPES:
            _check_input(x, what)
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.dim or (heads is not None and shape[1] != heads) or x.get_device() != self._index:
            raise ValueError(f"{what}: {name} must be [tokens, {'heads' if heads is None else heads}, {self.dim}] on {self.device}, got "
                             f"{tuple(shape)} on {x.device}")
        if x.is_contiguous():
            return x
        return x if x.stride(2) == 1 and x.stride(0) <= _STRIDE_MAX and x.stride(1) <= _STRIDE_MAX else x.contiguous()

    # -- tokens ------------------------------------------------------------------
    def append(self, layer: int, k: Tensor, v: Tensor, table: Tensor, lengths: Tensor, offsets: Optional[Tensor] = None) -> None:
        """Write new tokens' keys and values, ``k`` and ``v`` [tokens, kv_heads, dim] (bf16, fp16 or fp32).

        Rows ``offsets[b]`` .. ``offsets[b + 1] - 1`` (int32 [rows + 1]) are the last
        tokens of sequence b, whose ``lengths[b]`` counts them in already (``resize``'s ``ready``,
        where rows may have been refused); without ``offsets`` each sequence has one, and rows
        behind the last belong to none.  A page's scale is the least power of two, from 2^-48
        to 2^48, that takes the largest finite magnitude to 448 at most.  Tokens that join a
        page never make its scale smaller; where they make it larger, the codes that are there
        are rounded to it again.  Infinities and NaN become NaN codes.  Tokens whose place has
        no page in the table, or one that ``refs`` counts for more than one row, are not
        written: what other rows see is not changed.  No gradient: keys or values that want
        one, backward or forward, are refused.
        """
        what = "FP8KVCache.append"
        self._look()
        self._layer(what, layer)
        k, v = self._vectors(what, "k", k, self.kv_heads), self._vectors(what, "v", v, self.kv_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError(f"{what}: k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} do not fit")
        if _wants_derivative(k, v):
            raise RuntimeError(f"{what} has no gradient, backward or forward; pass detached keys and values")
        tokens = k.shape[0]
        (k_token, k_head, _), (v_token, v_head, _) = k.stride(), v.stride()
        table, rows, width, ld = self._table(what, table)
        lengths = self._ints(what, "lengths", lengths, (rows,))
        offsets = self._offsets(what, offsets, rows, tokens)
        dev = self.device
        need = 0 if offsets is None else _append_workspace(rows)
        work = _dense((need,), torch.uint8, dev) if need else None
        args = (self._ref, layer, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, _IN_DTYPES[k.dtype], tokens,
                table.data_ptr(), ld, width, lengths.data_ptr(), None if offsets is None else offsets.data_ptr(), rows,
                None if work is None else work.data_ptr(), need, _stream(dev))
        if self._index == _current_device():  # without a context, 0.2 us
            rc = _lib.lib().lrq_kv_append(*args)
        else:
            with _on(dev):
                rc = _lib.lib().lrq_kv_append(*args)
        if rc:
            _lib.check(rc, "lrq_kv_append")

    def attend(self, layer: int, q: Tensor, table: Tensor, lengths: Tensor, offsets: Optional[Tensor] = None, *,
               scale: Optional[float] = None, window: Optional[int] = None, out: Optional[Tensor] = None, return_lse: bool = False):
        """Causal attention of new tokens over their sequences' keys: ``q`` [tokens, heads, dim] (bf16 or fp16) -> the same.

        Tokens, ``lengths`` and ``offsets`` are as in ``append``, which goes before: a token
        sees its sequence's keys up to its own, the last ``window`` of them if that is
        given.  Query head i reads KV head ``i // (heads // kv_heads)``; ``scale`` is
        ``dim ** -0.5`` by default.  Scores and sums are float32, probabilities are rounded
        to fp16.  A token that sees no key gets 0; a NaN reaches the tokens that see it.
        Rows of no sequence (before the first one or behind the last) are 0, in a given ``out``
        (dense, of q's shape and type, q itself or apart from it) they stay as they are.
        ``return_lse`` adds the scores' log-sum-exp,
        float32 [tokens, heads] (-inf where nothing is seen).  No gradient: a backward
        pass through the result raises, and so does a ``q`` with a tangent.
        """
        what = "FP8KVCache.attend"
        self._look()
        q = self._vectors(what, "q", q, None)
        if q.dtype is torch.float32:
            raise TypeError(f"{what}: q must be bf16 or fp16")
        self._layer(what, layer)
        tokens, heads = q.shape[:2]
        if heads % self.kv_heads or not 1 <= heads <= 4096:
            raise ValueError(f"{what}: {heads} query heads (at most 4096) on {self.kv_heads} KV heads")
        if window is not None and (not isinstance(window, int) or window < 1):
            raise ValueError(f"{what}: window must be a whole number of at least 1, got {window!r}")
        scale = self.dim ** -0.5 if scale is None else float(scale)
        if not abs(scale) <= _SCALE_MAX:
            raise ValueError(f"{what}: scale {scale!r} (at most {_SCALE_MAX:.1e} in size)")
        table, rows, width, ld = self._table(what, table)
        lengths = self._ints(what, "lengths", lengths, (rows,))
        offsets = self._offsets(what, offsets, rows, tokens)
        if out is not None and (not isinstance(out, Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != self.device
                                or not out.is_contiguous() or out.data_ptr() % 8):
            raise ValueError(f"{what}: out must be a contiguous {tuple(q.shape)} {q.dtype} tensor on {self.device}, 8-byte aligned")
        args = (layer, q, table, ld, lengths, offsets, scale, min(window or 0, _WINDOW_MAX), out, return_lse)
        if _wants_derivative(q, q if out is None else out):
            if out is not None:
                raise RuntimeError(f"{what} has no gradient, backward or forward; pass no out, or a detached q")
            return NoGradient.apply(what, self._attend, *args)
        return self._attend(*args)

    def _attend(self, layer, q, table, ld, lengths, offsets, scale, window, out, return_lse):
        dev = self.device
        tokens, heads, dim = q.shape
        rows, width = table.shape
        given = out is not None
        if not given:
            out = _dense((tokens, heads, dim), q.dtype, dev)
        lse = _dense((tokens, heads), torch.float32, dev) if return_lse else None
        need = _attend_workspace(tokens, heads, self.kv_heads, dim, rows, offsets is None)
        work = _dense((need,), torch.uint8, dev)
        with _on(dev):
            rc = _lib.lib().lrq_kv_attend(self._ref, layer, q.data_ptr(), q.stride(0), q.stride(1), _IN_DTYPES[q.dtype], tokens, heads,
                                          table.data_ptr(), ld, width, lengths.data_ptr(),
                                          None if offsets is None else offsets.data_ptr(), rows, scale, window, not given,
                                          out.data_ptr(), None if lse is None else lse.data_ptr(), work.data_ptr(), need, _stream(dev))
        if rc:
            _lib.check(rc, "lrq_kv_attend")
        return (out, lse) if return_lse else out

    # -- pages -------------------------------------------------------------------
    def fork(self, table: Tensor, lengths: Tensor, parents: Tensor) -> tuple[Tensor, Tensor]:
        """Row r becomes row ``parents[r]`` (int32 [rows]) as it was: (new table, new lengths).

        The two rows share their pages, which ``refs`` counts; what row r held before is
        given back.  A row whose parent is itself, or no row, stays.  Entries behind a row's
        pages are -1.  The page that a sequence ends in stays shared until ``resize`` lets
        a row grow: resize before appending.
        """
        what = "FP8KVCache.fork"
        self._look()
        table, rows, width, ld = self._table(what, table)
        lengths = self._ints(what, "lengths", lengths, (rows,))
        parents = self._ints(what, "parents", parents, (rows,))
        dev = self.device
        out, out_lengths = _dense((rows, width), torch.int32, dev), _dense((rows,), torch.int32, dev)
        with _on(dev):
            rc = _lib.lib().lrq_kv_fork(self._ref, table.data_ptr(), ld, width, lengths.data_ptr(), rows, parents.data_ptr(),
                                        out.data_ptr(), out_lengths.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc, "lrq_kv_fork")
        return out, out_lengths

    def resize(self, table: Tensor, lengths: Tensor, wanted: Tensor, *, return_ready: bool = False) -> tuple[Tensor, ...]:
        """Pages for ``wanted`` tokens (int32 [rows]) in each row: (new table, new lengths, short).

        A row that shrinks gives back the pages behind its new end (all of them for 0).
        Rows that grow take the lowest free pages, in the rows' order; one that grows from
        inside a page which other rows hold too gets a copy of that page, in every layer (where
        all of its rows do, the last as well; the page itself is free after the call).
        Where free pages run out, counting what this call gives back, rows from there on that
        need any keep their length, and ``short`` (int32, no dimension) says how many pages
        were missing; a row that wants more than the table is wide keeps its length as well, and
        counts nothing there.  Entries behind a row's pages are -1.

        ``return_ready`` adds the lengths for this step's ``append`` and ``attend`` (int32
        [rows]): the new length of a row that has what it wanted, 0 of one that was refused.
        A row that gives tokens back and takes new ones in their place, in a page that others
        hold, is resized to what it keeps first.
        """
        what = "FP8KVCache.resize"
        self._look()
        table, rows, width, ld = self._table(what, table)
        lengths = self._ints(what, "lengths", lengths, (rows,))
        wanted = self._ints(what, "wanted", wanted, (rows,))
        dev = self.device
        out, out_lengths = _dense((rows, width), torch.int32, dev), _dense((rows,), torch.int32, dev)
        short = _dense((), torch.int32, dev)
        ready = _dense((rows,), torch.int32, dev) if return_ready else None
        need = _resize_workspace(rows, self.pages)
        work = _dense((need,), torch.uint8, dev)
        with _on(dev):
            rc = _lib.lib().lrq_kv_resize_ready(self._ref, table.data_ptr(), ld, width, lengths.data_ptr(), rows, wanted.data_ptr(),
                                                out.data_ptr(), out_lengths.data_ptr(), None if ready is None else ready.data_ptr(),
                                                short.data_ptr(), work.data_ptr(), need, _stream(dev))
        if rc:
            _lib.check(rc, "lrq_kv_resize_ready")
        return (out, out_lengths, short) if ready is None else (out, out_lengths, short, ready)

    def compact(self, table: Tensor) -> tuple[Tensor, Tensor]:
        """Move the pages in use together: (new table, their number n as an int32 without dimensions).

        Afterwards pages 0 .. n - 1 are in use.  The k-th page in use at or behind n moves,
        in every layer, to the k-th free one before n; ``refs`` follows.
        """
        what = "FP8KVCache.compact"
        self._look()
        table, rows, width, ld = self._table(what, table)
        dev = self.device
        out, count = _dense((rows, width), torch.int32, dev), _dense((), torch.int32, dev)
        need = _compact_workspace(self.pages)
        work = _dense((need,), torch.uint8, dev)
        with _on(dev):
            rc = _lib.lib().lrq_kv_compact(self._ref, table.data_ptr(), ld, width, rows, out.data_ptr(), count.data_ptr(),
                                           work.data_ptr(), need, _stream(dev))
        if rc:
            _lib.check(rc, "lrq_kv_compact")
        return out, count
