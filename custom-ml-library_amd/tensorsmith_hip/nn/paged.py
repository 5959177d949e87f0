"""A key/value cache held in 4 bits, in pages, and the attention that reads it.

Beside ``KVCache`` (one array, one length for all rows, 16 / 32 bits or int8): a
``PagedKVCache`` holds 4.5 bits a channel, its rows have lengths of their own, and a
row takes pages of ``page_size`` positions from a common pool as it grows.  Rows may
share pages -- beams, answers to one prompt -- until one of them appends into a
shared page, which is then copied for it.

The format (``include/tsattn.h``, ``tsattn_pages4``): e2m1 codes and a scale of 6
significant bits for each 32 channels, so that what the cache stands for is exact in
16 bits.  ``paged_attention`` reads the codes themselves for few query rows per KV
head, and for any number in fp32 or of 256 channels (``tsattn_pages4_attend``); for a
prompt's many rows of 16 bits the pages are dequantised once and attended as arrays.

Page tables and reference counts are the host's; lengths travel with each launch.
Calls captured into a HIP graph replay the positions, and the pages, that they were
captured at, so a replay is for as long as its rows keep both; a call that takes,
copies or gives back a page is refused there.  Calls on a cache and on its ``rows`` follow each
other: from several threads they take turns, and on another stream than the last
call's they wait for that stream (which has to live as long).  Replays are ordered by
who replays them.
"""

from __future__ import annotations

import math
import threading

import numpy as np

from .. import _lib
from ..device import device as parse_device
from ..device import _cuda, follow, state
from ..tensor import Tensor, backend_dtype, is_grad_enabled, to_numpy
from .attention import _dtype_code, _rope_rows, rope_tables, scaled_dot_product_attention


def _reads_codes(rows: int, heads: int, dim: int, wide: bool, lens) -> bool:
    """Whether attention reads the codes themselves: ``rows`` query rows per KV head over sequences
    of ``lens``.  Dequantising once costs host time for each run of rows of one length, and memory
    traffic, and has the faster matrix products afterwards; of fp32 (``wide``) it has not: three bf16
    parts take a seventh of the fp32 kernels' time.  Microseconds, codes / dequantised, 8 KV heads of
    D128, bf16: over 8000 positions 128 rows 28 / 50, 256 48 / 51, 512 65 / 50, 1024 119 / 59; over
    2000, 1024 rows 36 / 50, 2048 60 / 50; 4 sequences of 8000, 128 rows 72 / 122, 512 224 / 120; 8
    heads of D64, 2 of 2000, 1024 rows 38 / 50, 2048 64 / 45.  fp32, 8 heads of D128 over 8000: 1024
    rows 158 / 1135.  Not for more rows than the codes' kernel takes, nor where its splits of 4096
    positions would leave more than 4 GiB of partial sums (of positions that are there: the scratch
    goes by the longest row, and is bounded by the library, which takes a call in parts).  The two
    keep P in different bits: the codes' kernel in two or three bf16 parts, within 2^-16 of it or
    exactly, the kernels of arrays in the dtype (bf16 2^-8, f16 2^-11: the matrix cores' operand)."""
    if rows > 1 << 18 or 4 * rows * heads * dim * int((-(-lens // 4096)).sum()) > 1 << 32:
        return False
    pairs, size = rows * heads * int(lens.sum()), (dim / 128) ** 0.85
    codes = 15 + 1.8e-6 * size * pairs
    whole = 42 * len(_runs(lens)) + 1.5e-6 * dim * heads * int(lens.sum()) + 4e-7 * size * pairs
    return wide or codes <= whole


def _runs(lens) -> list:
    """Ends of the runs of rows of one length."""
    return [*(np.flatnonzero(lens[1:] != lens[:-1]) + 1).tolist(), len(lens)]


def _rows(t):
    """``t`` with rows that the kernels read as they are: 16-byte aligned, channels side by side."""
    import torch

    a, b, c, d = t.stride()
    if d == 1 and not (a | b | c) & 7 and not t.data_ptr() & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _view(t) -> _lib.View:
    v = _lib.View()
    v.data = t.data_ptr()
    v.stride[:] = t.stride()
    return v


class _Pages:
    """The pool, the page table (host and device) and the rows' lengths.  Pages are given out and
    taken back by the library's host calls over these arrays (``tsattn_pages4_host``)."""

    def __init__(self, rows: int, heads: int, dim: int, columns: int, page_size: int, num_pages: int, dev):
        import torch

        self.heads, self.dim, self.page_size, self.device = heads, dim, page_size, dev
        self.lock = threading.RLock()  # (a call's changes, its update and its launch belong together)
        self.page_bytes = int(_lib.load().tsattn_pages4_page_bytes(heads, page_size, dim))
        if not self.page_bytes:
            raise NotImplementedError("paged caches take head dims 32, 64, 128 and 256, up to 4096 heads and "
                                      "pages of 32, 64, .. 4096 positions")
        # the host's arrays, side by side; src, dst: page copies that a call asks for; some: lengths or
        # positions of a call's rows
        most, entries = max(rows, num_pages), rows * columns
        sizes = {"host": entries, "lengths": rows, "refs": num_pages, "stack": num_pages, "shown": entries,
                 "changed": entries, "src": most, "dst": most, "copies": 1, "some": rows, "dirty": (entries + 3) // 4}
        memory, at, where, part = np.zeros(sum(sizes.values()), np.int32), 0, {}, {}
        base = memory.ctypes.data
        for name, n in sizes.items():
            part[name], where[name] = memory[at:at + n], base + 4 * at
            at += n
        self.host, self.lengths, self.refs = part["host"].reshape(rows, columns), part["lengths"], part["refs"]
        self.stack, self.shown, self.copies = part["stack"], part["shown"], part["copies"]
        self.lengths_at, self.some, self.some_at = where["lengths"], part["some"], where["some"]
        # the stream of the call at hand, and of the last one that was not captured; where it may change
        # pages, whether its device is current, and whether it is captured
        self.now, self.stream = follow(dev)
        self.here = self.captured = False
        self.pending = False  # whether page copies or entries may be left to bring to the device
        self.out = where["src"], where["dst"], where["copies"]
        self.tables = _lib.Pages4Host(rows, columns, page_size, num_pages, where["host"], where["lengths"], where["refs"],
                                      where["stack"], where["shown"], where["changed"], where["dirty"], 0, 0)
        # (what no append has written weighs nothing: positions past a row's length are masked)
        self.pool = torch.empty((num_pages, self.page_bytes), dtype=torch.uint8, device=dev.torch)
        self.table = torch.empty((rows, columns), dtype=torch.int32, device=dev.torch)
        self.desc = _lib.Pages4(self.pool.data_ptr(), num_pages, heads, page_size, dim, self.table.data_ptr(), rows,
                                columns)

    def clear(self) -> None:
        """Every page free, every row empty."""
        pages = len(self.refs)
        self.host.fill(-1)
        self.shown.fill(-1)
        self.stack[:] = np.arange(pages - 1, -1, -1)  # (the next one is the last)
        self.tables.free = pages

    @property
    def free(self) -> int:
        return self.tables.free

    def ready(self, changes: bool = False) -> None:
        """Every call begins with it: what was queued before on another stream comes first (a page that
        is given back and taken again may still be read there), and what an earlier call's page
        changes left to do, if it failed before they were on the device.  ``changes``: the call may
        change pages."""
        self.now, self.stream = follow(self.device, self.stream, self.pool, self.table)
        self.here, self.captured = state(self.device) if changes or self.pending else (False, False)
        if self.pending:
            if self.copies[0] or self.tables.n_changed:
                self._eager()
            self.apply()

    def call(self, function, *args) -> int:
        """``device.launch``, on the stream that ``ready`` found."""
        if self.here or _cuda().current_device() == self.device.index:
            return function(*args, self.now)
        with _cuda().device(self.device.index):
            return function(*args, self.now)

    def apply(self, source=None) -> None:
        """To the device, on the current stream: the page copies that the last host call asked for
        (from the pool of ``source``, by default this one's) and the changed table entries."""
        n = int(self.copies[0])
        if n or self.tables.n_changed:
            pool = (source or self).desc
            _lib.check(self.call(_lib.load().tsattn_pages4_apply, self.tables, self.desc.table, pool.pool,
                                 pool.num_pages, self.desc.pool, self.desc.num_pages, self.page_bytes, n,
                                 *self.out[:2]), "page update")
            self.copies[0] = 0
        self.pending = False

    def _eager(self, rows=None, steps: int = 0) -> None:
        """Refuses page changes under capture: a captured call's pages would be the host's at once and
        the device's with each replay.  With ``rows``: only if they need other pages for ``steps``."""
        if not self.captured:
            return
        if rows is not None:
            lens = self.lengths[rows]
            page = self.host[rows, lens // self.page_size % self.host.shape[1]]
            part = lens % self.page_size
            if ((part > 0) & (part + steps <= self.page_size) & (self.refs[np.maximum(page, 0)] == 1)).all():
                return
        raise RuntimeError("a paged cache's pages cannot change while a graph is captured")

    def grow(self, n: int, rows: int, steps: int) -> None:
        """Pages of their own for the next ``steps`` positions of the ``n`` rows (an address)."""
        self.pending = True
        _lib.check(_lib.load().tsattn_pages4_grow(self.tables, n, rows, steps, *self.out), "page table")

    def cut(self, rows, rows_at: int, lengths=0) -> None:
        """``rows`` (at an address) end at ``lengths``; pages wholly past them are given back (under
        capture refused: the captured calls would go on with them)."""
        self.ready(True)
        to = self.some[:len(rows)]
        to[:] = lengths
        if (to != lengths).any():  # (more than 32 bits)
            raise ValueError("truncate length must be between zero and the current length")
        if self.captured:
            pages = -(-self.lengths[rows] // self.page_size)
            if ((to >= 0) & (-(-to // self.page_size) < pages)).any():
                self._eager()
        _lib.check(_lib.load().tsattn_pages4_cut(self.tables, len(rows), rows_at, self.some_at), "page table")

    def take_back(self, rows, steps: int) -> None:
        """Gives back the pages that ``grow`` took past the rows' lengths, if it got so far.  Copies of
        shared pages stay: they are the rows' own, made with the next call if they are not there yet."""
        held = ((self.host[rows] >= 0).sum(1) * self.page_size).astype(np.int32)
        lens = self.lengths[rows]
        self.lengths[rows] = np.maximum(lens, np.minimum(lens + np.int32(steps), held))
        _lib.check(_lib.load().tsattn_pages4_cut(self.tables, len(rows), rows.ctypes.data, lens.ctypes.data), "page table")

    def clone(self, rows, num_pages: int) -> "_Pages":
        """The rows with pages of their own, in a pool of ``num_pages``."""
        self.ready(True)
        self._eager()
        other = _Pages(len(rows), self.heads, self.dim, self.host.shape[1], self.page_size, num_pages, self.device)
        _lib.check(_lib.load().tsattn_pages4_clone(self.tables, len(rows), rows.ctypes.data, other.tables, *other.out),
                   "page table")
        other.apply(self)
        return other


class PagedKVCache:
    """4-bit keys and values of ``batch_size`` sequences of up to ``max_seq_len`` positions.

    ``num_pages`` pages of ``page_size`` (32, 64, 128, .. 4096) positions are
    allocated at once; by default as many as the rows can need.  ``dtype`` (float32,
    float16 or bfloat16) is that of the keys and values given and read back.
    Inference only, like ``KVCache``.  Where a launch fails, ``append`` leaves the rows as
    they were; ``reorder`` and ``compact`` have taken place on the host, and the next call
    first brings to the device what it lacks.
    """

    def __init__(self, batch_size: int, num_heads: int, head_dim: int, max_seq_len: int, *, device=None,
                 dtype="float32", page_size: int = 64, num_pages: int | None = None):
        if min(batch_size, num_heads, head_dim, max_seq_len, page_size) <= 0:
            raise ValueError("cache dimensions and capacity must be positive")
        dev = parse_device(device)
        if dev.type != "hip":
            raise RuntimeError("tensorsmith_hip keeps KV caches on hip devices")
        self.dtype = backend_dtype(dtype, dev)
        if str(self.dtype).split(".")[-1] not in ("float32", "float16", "bfloat16"):
            raise TypeError("paged caches hold float32, float16 or bfloat16 rows")
        columns = -(-max_seq_len // page_size)
        if num_pages is None:
            num_pages = batch_size * columns
        if num_pages <= 0:
            raise ValueError("cache dimensions and capacity must be positive")
        self.max_seq_len, self._code = max_seq_len, _dtype_code(self.dtype)
        self._core = _Pages(batch_size, num_heads, head_dim, columns, page_size, num_pages, dev)
        self._core.clear()
        self._select()

    def _select(self, rows=None) -> None:
        """The core's rows that this cache is; all of them by default."""
        every = len(self._core.lengths)
        self._whole = rows is None or (len(rows) == every and bool((rows == np.arange(every)).all()))
        self._rows = np.arange(every, dtype=np.int32) if rows is None else rows
        self._rows_at = self._rows.ctypes.data

    # -- what it is -----------------------------------------------------------

    batch_size = property(lambda self: len(self._rows))
    num_heads = property(lambda self: self._core.heads)
    head_dim = property(lambda self: self._core.dim)
    value_dim = head_dim
    device = property(lambda self: self._core.device)
    page_size = property(lambda self: self._core.page_size)
    num_pages = property(lambda self: self._core.pool.shape[0])
    quantized = True

    @property
    def lengths(self) -> tuple:
        """Cached positions of every row."""
        return tuple(self._core.lengths[self._rows].tolist())

    @property
    def length(self) -> int:
        """Cached positions of the longest row."""
        return int(self._core.lengths[self._rows].max())

    @property
    def pages_in_use(self) -> int:
        return self.num_pages - self._core.free

    @property
    def memory_bytes(self) -> int:
        """Allocated persistent payload: the pool and its table."""
        return self._core.pool.numel() + 4 * self._core.table.numel()

    def __len__(self):
        return self.length

    def __repr__(self):
        return (f"PagedKVCache(rows={self.batch_size}, length={self.length}, capacity={self.max_seq_len}, "
                f"pages={self.pages_in_use}/{self.num_pages}, device='{self.device}')")

    # -- rows in and out ------------------------------------------------------

    def append(self, key: Tensor, value: Tensor, *, rotary_base: float | None = None) -> None:
        """Quantise and append ``key`` and ``value`` [B, H, T, D], each row at its own length.

        ``rotary_base``: rotate the keys by RoPE at those positions first, as
        ``rotary_embedding`` does.  Nothing changes if the pool has too few free pages.
        """
        self._check(key, value)
        core, steps = self._core, key._data.shape[2]
        with core.lock:
            lens, lens_at = self._lens()
            most = int(lens.max()) + steps
            if steps == 0 or most > self.max_seq_len:
                raise ValueError(f"cache capacity {self.max_seq_len} exceeded or empty append")
            cos = sin = None
            if rotary_base is not None:
                if rotary_base <= 0 or not math.isfinite(rotary_base):
                    raise ValueError("RoPE requires a positive even rotary dimension and valid positions/base")
                cos, sin = (t.data_ptr() for t in rope_tables(rotary_base, core.dim, self.dtype, core.pool.device, most))
            k, v = (_rows(t if t.dtype == self.dtype else t.to(self.dtype)) for t in (key._data, value._data))
            core.ready(True)
            if core.captured:
                core._eager(self._rows, steps)
            try:
                core.grow(len(lens), self._rows_at, steps)
                core.apply()
                _lib.check(core.call(_lib.load().tsattn_pages4_append, core.desc, self._code, len(lens), steps,
                                     _view(k), _view(v), self._rows_at, lens_at, cos, sin), "paged append")
            except BaseException:
                core.take_back(self._rows, steps)
                raise
            if self._whole:
                core.lengths += steps
            else:
                core.lengths[self._rows] += steps

    def _lens(self):
        """The rows' lengths and their address."""
        if self._whole:
            return self._core.lengths, self._core.lengths_at
        lens = self._core.lengths[self._rows]
        return lens, lens.ctypes.data

    def _check(self, key: Tensor, value: Tensor) -> None:
        """``KVCache``'s refusals, in its order."""
        dev = self._core.device
        if (key.device is not dev and key.device != dev) or (value.device is not dev and value.device != dev):
            raise ValueError("cache and key/value tensors must be on the same device")
        if (key.requires_grad or value.requires_grad) and is_grad_enabled():
            raise RuntimeError("KVCache is inference-only; use no_grad() for differentiable inputs")
        shape = tuple(key._data.shape)
        if len(shape) != 4 or shape[:2] != (len(self._rows), self._core.heads) or shape[3] != self._core.dim:
            raise ValueError("key shape does not match cache configuration")
        if tuple(value._data.shape) != shape:
            raise ValueError("value shape does not match cache configuration")

    def get(self, last: int | None = None) -> tuple[Tensor, Tensor]:
        """Keys and values as they are held [B, H, T, D]: all positions up to the longest
        row's length (zero past a row's own), or the ``last`` positions of every row."""
        import torch

        core = self._core
        with core.lock:
            core.ready()
            lens, lens_at = self._lens()
            if last is not None and not 0 < last <= lens.min():
                raise ValueError("the last positions read must be between one and the shortest row's length")
            steps = int(lens.max()) if last is None else last
            first = core.some[:len(lens)]
            if last is None:
                first[:] = 0
            else:
                np.subtract(lens, last, out=first)
            k = torch.empty((len(lens), core.heads, steps, core.dim), dtype=self.dtype, device=core.pool.device)
            v = torch.empty_like(k)
            if steps:
                _lib.check(core.call(_lib.load().tsattn_pages4_read, core.desc, self._code, len(lens), steps,
                                     _view(k), _view(v), self._rows_at, lens_at, core.some_at), "paged read")
        return Tensor._leaf(k, core.device), Tensor._leaf(v, core.device)

    # -- rows and pages -------------------------------------------------------

    def rows(self, indices) -> "PagedKVCache":
        """These rows as a cache of their own over the same pages: to fill a row that was
        freed, or to step some rows alone.  Both change together."""
        index = self._indices(indices, None)
        if len(index) == 0 or len(np.unique(index)) != len(index):
            raise ValueError("rows must be different and at least one")
        view = object.__new__(PagedKVCache)
        view.dtype, view.max_seq_len, view._code, view._core = self.dtype, self.max_seq_len, self._code, self._core
        view._select(np.ascontiguousarray(self._rows[index]))
        return view

    def _indices(self, indices, shape):
        host = np.asarray(to_numpy(indices._data) if isinstance(indices, Tensor) else indices)
        if host.ndim != 1 or (shape is not None and host.shape != shape) or (host.size and host.dtype.kind not in "iu"):
            raise ValueError("beam indices must be one integer per cache batch row" if shape is not None
                             else "row indices must be integers")
        index = host.astype(np.int32)
        if shape is None and index.size and (index.min() < 0 or index.max() >= len(self._rows)) or (index != host).any():
            raise ValueError("beam index out of range" if shape is not None else "row index out of range")
        return index  # (a beam index's range is checked with the tables)

    def reset(self) -> None:
        """Every row empty, its pages given back."""
        with self._core.lock:
            self._core.cut(self._rows, self._rows_at)

    def free(self, indices) -> None:
        """These rows empty, their pages given back."""
        rows = self._rows[np.unique(self._indices(indices, None))]
        if len(rows):
            with self._core.lock:
                self._core.cut(rows, rows.ctypes.data)

    def truncate(self, length) -> None:
        """Cut every row to ``length`` positions, or to a length of its own (a sequence of them);
        pages wholly past it are given back."""
        want = np.asarray(length)
        if want.dtype.kind not in "iu" or want.shape not in ((), self._rows.shape):
            raise ValueError("truncate takes one integer length, or one per row")
        with self._core.lock:
            self._core.cut(self._rows, self._rows_at, want)

    def reorder(self, indices) -> None:
        """Row i becomes row ``indices[i]``, sharing its pages: no keys or values move.  Rows that
        take over the same row share until one appends (``append`` copies the page)."""
        core, index = self._core, self._indices(indices, self._rows.shape)
        with core.lock:
            core.ready(True)
            core._eager()
            core.pending = True
            _lib.check(_lib.load().tsattn_pages4_reorder(core.tables, len(index), self._rows_at, index.ctypes.data),
                       "page table")
            core.apply()

    def copy(self, num_pages: int | None = None) -> "PagedKVCache":
        """A cache of these rows with a pool of its own (``num_pages``, by default as many as this
        one has), its pages in use side by side; rows that share pages share them there."""
        other = object.__new__(PagedKVCache)
        other.dtype, other.max_seq_len, other._code = self.dtype, self.max_seq_len, self._code
        with self._core.lock:
            other._core = self._core.clone(self._rows, self._pool_size(num_pages))
        other._select()
        return other

    def compact(self, num_pages: int | None = None) -> int:
        """Move the pages in use to the front of the pool, and with ``num_pages`` into a pool of that
        size (smaller or larger); returns how many are in use."""
        core = self._core
        with core.lock:
            if num_pages is None:
                core.ready(True)
                core._eager()
                core.pending = True
                _lib.check(_lib.load().tsattn_pages4_compact(core.tables, *core.out), "page table")
                core.apply()
            else:
                new = core.clone(np.arange(len(core.lengths), dtype=np.int32), self._pool_size(num_pages))
                core.__dict__.update({**new.__dict__, "lock": core.lock})
            return self.pages_in_use

    def _pool_size(self, num_pages) -> int:
        """``num_pages``, by default as many as there are; refused if fewer than are in use here."""
        if num_pages is None:
            return self.num_pages
        rows = self._core.host if self._whole else self._core.host[self._rows]
        used = len(np.unique(rows[rows >= 0]))
        if num_pages < max(used, 1):
            raise ValueError(f"{used} pages are in use")
        return num_pages


def paged_attention(query: Tensor, cache: PagedKVCache, *, is_causal: bool = True, scale: float | None = None,
                    rotary_base: float | None = None) -> Tensor:
    """Attention of ``query`` [B, Hq, T, D] over a ``PagedKVCache``'s rows.

    The queries are at the last T positions of their row (append their keys and values
    first): with ``is_causal`` each sees the positions up to its own, else all.  Query
    heads may be a multiple of the cache's.  ``rotary_base`` rotates the queries by
    RoPE at those positions.  A query that sees nothing gives zero.  Inference only.
    """
    core, q = cache._core, query._data
    if query.ndim != 4:
        raise ValueError("attention expects [batch, heads, sequence, channels]")
    if query.device is not core.device and query.device != core.device:
        raise ValueError("attention tensors must be on the same device")
    if q.dtype != cache.dtype:
        raise TypeError("attention inputs must have the same floating-point dtype")
    b, heads, steps, dim = q.shape
    if b != len(cache._rows) or dim != core.dim:
        raise ValueError("query shape does not match cache configuration")
    if not heads or not steps or heads % core.heads:
        raise ValueError("grouped-query attention requires enable_gqa and query heads divisible by KV heads")
    if query.requires_grad and is_grad_enabled():
        raise RuntimeError("KVCache is inference-only; use no_grad() for differentiable inputs")
    multiplier = 1 / math.sqrt(dim) if scale is None else scale
    if not math.isfinite(multiplier):
        raise ValueError("attention scale must be finite")
    if rotary_base is not None and (rotary_base <= 0 or not math.isfinite(rotary_base)):
        raise ValueError("RoPE requires a positive even rotary dimension and valid positions/base")
    import torch

    with core.lock:
        core.ready()
        lens, lens_at = cache._lens()
        rows = heads // core.heads * steps
        if (rows > 32 and dim <= 128 and lens.min() >= steps
                and not _reads_codes(rows, core.heads, dim, q.dtype == torch.float32, lens)):
            return _prompt(query, cache, lens, is_causal, multiplier, rotary_base)
        q = _rows(q)
        cos = sin = None
        if rotary_base is not None:
            cos, sin = (t.data_ptr() for t in rope_tables(rotary_base, dim, q.dtype, q.device,
                                                          max(int(lens.max()), steps)))
        out = torch.empty((b, heads, steps, dim), dtype=q.dtype, device=q.device)
        lib, code = _lib.load(), cache._code
        nbytes = lib.tsattn_pages4_attend_workspace(core.desc, code, b, heads, steps, lens_at)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _lib.check(core.call(lib.tsattn_pages4_attend, core.desc, code, b, heads, steps, multiplier,
                             int(is_causal), _view(q), _view(out), cache._rows_at, lens_at, cos, sin,
                             None if ws is None else ws.data_ptr(), nbytes), "paged attention")
    return Tensor._from_op(out, (query,), None, "paged_attention")


def _prompt(query: Tensor, cache: PagedKVCache, lens, is_causal: bool, scale: float, rotary_base) -> Tensor:
    """Many query rows: the values dequantised once, then the attention of arrays; runs of rows of
    one length one after the other."""
    import torch

    def attend(q, held, n):
        if rotary_base is not None:
            q = _rope_rows(q, n - q.shape[2], rotary_base, q.shape[3], False, cache.device)
        k, v = held.get()
        return scaled_dot_product_attention(
            Tensor(q, device=cache.device), k, v, None, 0.0, is_causal, scale=scale,
            causal_offset=n - q.shape[2] if is_causal else 0, enable_gqa=q.shape[1] != held.num_heads)._data

    q, parts, first = query._data, [], 0
    with torch.cuda.device(cache.device.index):  # (attention launches on the current device)
        for stop in _runs(lens):
            held = cache if stop - first == len(lens) else cache.rows(range(first, stop))
            parts.append(attend(q[first:stop], held, int(lens[first])))
            first = stop
    out = parts[0] if len(parts) == 1 else torch.cat(parts)
    return Tensor._from_op(out, (query,), None, "paged_attention")
