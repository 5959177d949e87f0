"""The paged 4-bit cache on the host: page tables, reference counts and copies on
write against rows kept as lists, and the refusals of both interfaces.

The kernels stand in as functions over CPU memory that keep a tag a position: what
they are told to copy, set and append has to leave every row its own tags.
"""

from __future__ import annotations

import ctypes
import gc
import importlib
import random
import weakref
from contextlib import ExitStack, nullcontext
from unittest.mock import patch

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tensorsmith_hip as ts  # noqa: E402
from tensorsmith_hip import _lib, nn  # noqa: E402

D = importlib.import_module("tensorsmith_hip.device")
P = importlib.import_module("tensorsmith_hip.nn.paged")


REAL = _lib.load()


def _at(address, n, kind):
    address = getattr(address, "value", address)
    return np.frombuffer((ctypes.c_char * (n * np.dtype(kind).itemsize)).from_address(address), kind)


class Memory:
    """The entry points over CPU memory: a page is one float64 tag a position."""

    def __init__(self):
        self.calls, self.fail = [], False

    def __getattr__(self, name):  # the calls that change the host's tables alone
        assert name in ("tsattn_pages4_" + x for x in ("grow", "cut", "reorder", "clone", "compact")), name
        return getattr(REAL, name)

    def tsattn_pages4_page_bytes(self, heads, page, dim):
        return page * 8 if dim in (32, 64, 128, 256) else 0

    def tsattn_pages4_apply(self, host, table, source, sn, target, tn, page_bytes, n, src, dst, stream):
        if n:
            src, dst = _at(src, n, np.int32), _at(dst, n, np.int32)
            assert len(set(dst)) == n and (source != target or not set(dst) & set(src))
            old, new = (_at(x, m * page_bytes, np.uint8).reshape(m, -1) for x, m in ((source, sn), (target, tn)))
            new[dst] = old[src]
            self.calls.append(("copy", n))
        entries = host.rows * host.columns
        at, want = _at(host.changed, entries, np.int32)[:host.n_changed], _at(host.table, entries, np.int32)
        assert len(set(at)) == len(at) and _at(host.dirty, entries, np.uint8).sum() == len(at)
        assert _at(host.dirty, entries, np.uint8)[at].all()
        shown = _at(host.shown, entries, np.int32)
        at = at[(want[at] >= 0) & (want[at] != shown[at])]
        _at(table, entries, np.int32)[at] = shown[at] = want[at]
        _at(host.dirty, entries, np.uint8)[:] = 0
        host.n_changed = 0
        if len(at):
            self.calls.append(("set", len(at)))
        return 0

    def tsattn_pages4_append(self, desc, dtype, n, steps, k, v, rows, lens, cos, sin, stream):
        if self.fail:
            return _lib.ERR_HIP
        table = _at(desc.table, desc.table_rows * desc.table_stride, np.int32).reshape(desc.table_rows, -1)
        pool = _at(desc.pool, desc.num_pages * desc.page_size, np.float64).reshape(desc.num_pages, -1)
        for i, (row, length) in enumerate(zip(_at(rows, n, np.int32), _at(lens, n, np.int32))):
            for t in range(steps):
                tag = _at(k.data + 4 * (i * k.stride[0] + t * k.stride[2]), 1, np.float32)[0]
                pool[table[row, (length + t) // desc.page_size], (length + t) % desc.page_size] = tag
        self.calls.append(("append", steps))
        return 0


@pytest.fixture
def memory():
    memory = Memory()
    with ExitStack() as stack:
        for patched in (patch.object(D.Device, "torch", torch.device("cpu")),
                        patch.object(D, "is_available", lambda value: True),
                        patch.object(D, "current_stream", lambda dev: 0),
                        patch.object(torch.cuda, "current_device", lambda: 0),
                        patch.object(torch.cuda, "is_current_stream_capturing", lambda: False),
                        patch.object(torch.cuda, "device", lambda index: nullcontext()),
                        patch.object(_lib, "load", lambda: memory),
                        patch.object(_lib, "last_error", lambda: REAL.tsattn_last_error().decode())):
            stack.enter_context(patched)
        yield memory


def _held(cache, row):
    core = cache._core
    pool = core.pool.numpy().view(np.float64).reshape(core.pool.shape[0], -1)
    table = core.table.numpy()
    n = core.lengths[row]
    return [pool[table[row, p // core.page_size], p % core.page_size] for p in range(n)]


def _sound(cache, want):
    core = cache._core
    held = core.host >= 0
    assert core.tables.n_changed == 0 and (core.table.numpy()[held] == core.host[held]).all() and (core.shown.reshape(core.host.shape)[held] == core.host[held]).all()
    used = core.host[core.host >= 0]
    assert (np.bincount(used, minlength=len(core.refs)) == core.refs).all()
    free = core.stack[:core.free]
    assert len(set(free.tolist())) == core.free and not set(free.tolist()) & set(used.tolist())
    assert core.free + len(set(used.tolist())) == len(core.refs) == cache.num_pages
    assert list(cache.lengths) == [len(x) for x in want]
    assert (core.host >= 0).sum(1).tolist() == [-(-len(x) // core.page_size) for x in want]
    for row, tags in enumerate(want):
        assert _held(cache, row) == tags, row


def _rows(tags):
    """Keys (and values) whose first channel is the tag: tags [B][T]."""
    x = torch.zeros(len(tags), 2, len(tags[0]), 32)
    x[:, :, :, 0] = torch.tensor(tags, dtype=torch.float32)[:, None]
    return ts.Tensor(x, device="hip")


@pytest.mark.parametrize("seed", range(12))
def test_rows_keep_their_own_positions(memory, seed):
    """Random appends, forks, cuts, frees and moves; a pool that sometimes runs out."""
    rng = random.Random(seed)
    b, most, page = rng.choice([1, 3, 5]), rng.choice([150, 400]), rng.choice([32, 64])
    full = b * -(-most // page)
    cache = nn.PagedKVCache(b, 2, 32, most, device="hip", page_size=page,
                            num_pages=rng.choice([full, full, max(2, full * 2 // 3)]))
    want, tag = [[] for _ in range(b)], [1.0]

    def fresh(rows, n):
        out = [[tag[0] + i * n + j for j in range(n)] for i in range(rows)]
        tag[0] += rows * n
        return out

    for _ in range(60):
        what = rng.choice(["append"] * 5 + ["some", "reorder", "truncate", "cut", "free", "compact", "resize", "copy"])
        if what in ("append", "some"):
            index = list(range(b)) if what == "append" else rng.sample(range(b), rng.randint(1, b))
            n = rng.choice([1, 1, 1, 2, rng.randint(1, 90)])
            if max(len(want[i]) for i in index) + n > most:
                continue
            new, target = fresh(len(index), n), cache if what == "append" else cache.rows(index)
            try:
                target.append(_rows(new), _rows(new))
            except ValueError as error:
                assert "pool exhausted" in str(error)
            else:
                for i, x in zip(index, new):
                    want[i] = want[i] + x
        elif what == "reorder":
            index = [rng.randrange(b) for _ in range(b)]
            memory.calls.clear()
            cache.reorder(index)
            assert not any(name == "copy" for name, _ in memory.calls)
            want = [list(want[i]) for i in index]
        elif what == "truncate":
            n = rng.randint(0, min(len(x) for x in want))
            cache.truncate(n)
            want = [x[:n] for x in want]
        elif what == "cut":
            lens = [max(0, len(x) - rng.choice([0, 1, 40])) for x in want]
            cache.truncate(lens)
            want = [x[:n] for x, n in zip(want, lens)]
        elif what == "free":
            index = rng.sample(range(b), rng.randint(0, b))
            cache.free(index)
            want = [[] if i in index else x for i, x in enumerate(want)]
        elif what == "compact":
            assert cache.compact() == cache.pages_in_use
            assert cache._core.host.max() < max(cache.pages_in_use, 1)
        elif what == "resize":
            n = cache.pages_in_use + rng.choice([0, 1, full])
            cache.compact(max(n, 1))
            assert cache.num_pages == max(n, 1)
        else:
            other = cache.copy()
            _sound(other, want)
            if b and max(len(x) for x in want) < most and other.pages_in_use + 2 * b <= other.num_pages:
                other.append(_rows(fresh(b, 1)), _rows(fresh(b, 1)))  # its pages are its own
        _sound(cache, want)


def test_beams_copy_one_page_each(memory):
    """Eight rows of one prompt: no copies until they append, then all but one copy its last page once."""
    cache = nn.PagedKVCache(8, 2, 32, 300, device="hip", page_size=64)
    cache.rows([0]).append(_rows([[float(i) for i in range(100)]]), _rows([[0.0] * 100]))
    cache.reorder([0] * 8)
    assert cache.pages_in_use == 2 and cache.lengths == (100,) * 8
    memory.calls.clear()
    cache.append(_rows([[1000.0 + i] for i in range(8)]), _rows([[0.0]] * 8))
    assert ("copy", 7) in memory.calls and cache.pages_in_use == 1 + 8
    memory.calls.clear()
    for _ in range(26):  # up to and past the page's end: no more copies
        cache.append(_rows([[1.0]] * 8), _rows([[1.0]] * 8))
    assert not any(name == "copy" for name, _ in memory.calls)
    # positions 102 .. 127 touch no page but their own: nothing but the append is called
    assert {name for name, _ in memory.calls} == {"append"}


def test_rows_that_grow_or_fork_again_find_their_pages(memory):
    """Drafted tokens that are dropped change no table entry; beams that start over, no more than their own."""
    cache = nn.PagedKVCache(4, 2, 32, 300, device="hip", page_size=32)
    cache.append(_rows([[0.0] * 100] * 4), _rows([[0.0] * 100] * 4))
    cache.truncate([64, 65, 90, 32])
    for _ in range(3):
        cache.append(_rows([[1.0] * 70] * 4), _rows([[1.0] * 70] * 4))
        cache.truncate([64, 65, 90, 32])
    memory.calls.clear()
    cache.append(_rows([[1.0] * 70] * 4), _rows([[1.0] * 70] * 4))
    assert [x for x in memory.calls if x[0] == "set"] == []
    for i in range(3):
        memory.calls.clear()
        cache.truncate([40] * 4 if i else [40, 64, 64, 64])
        cache.reorder([0] * 4)
        cache.append(_rows([[2.0]] * 4), _rows([[2.0]] * 4))
        assert ("copy", 3) in memory.calls
    assert [n for name, n in memory.calls if name == "set"] == [3, 3]  # the shared page, and back


@pytest.mark.parametrize("index", [0, 1])
def test_calls_launch_on_the_caches_device(memory, index):
    """With the cache's device current, on its current stream, whichever was current before."""
    seen, state = [], {"device": 0}

    class on:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.before, state["device"] = state["device"], self.device

        def __exit__(self, *_):
            state["device"] = self.before

    class Noting:
        def __getattr__(self, name):
            if name == "tsattn_pages4_attend_workspace":
                return lambda *a: 64
            launches = name in ("tsattn_pages4_" + x for x in ("append", "apply", "read", "attend"))
            call = (lambda *a: 0) if name.endswith(("read", "attend")) else getattr(memory, name)
            return lambda *a: (launches and seen.append((name, state["device"], a[-1]))) or call(*a)

    with patch.object(torch.cuda, "current_device", lambda: state["device"]), patch.object(torch.cuda, "device", on), \
            patch.object(D, "current_stream", lambda dev: 0x100 + dev.index), patch.object(_lib, "load", lambda: Noting()):
        dev = f"hip:{index}"
        x = lambda *s: ts.Tensor(torch.zeros(s), device=dev)  # noqa: E731
        cache = nn.PagedKVCache(2, 2, 32, 100, device=dev)
        cache.append(x(2, 2, 3, 32), x(2, 2, 3, 32), rotary_base=100.0)
        cache.reorder([1, 1])
        cache.append(x(2, 2, 1, 32), x(2, 2, 1, 32))
        cache.get(), cache.copy(), cache.compact(7)
        nn.paged_attention(x(2, 4, 1, 32), cache, rotary_base=100.0)
        with pytest.raises(ValueError, match="same device"):
            other = ts.Tensor(torch.zeros(2, 4, 1, 32), device=f"hip:{1 - index}")
            nn.paged_attention(other, cache)
    assert {name for name, _, _ in seen} == {"tsattn_pages4_" + x for x in ("append", "apply", "read", "attend")}
    assert all(device == index and stream == 0x100 + index for _, device, stream in seen), seen
    assert state["device"] == 0


def test_a_failed_append_leaves_the_lengths(memory):
    cache = nn.PagedKVCache(2, 2, 32, 100, device="hip")
    cache.append(_rows([[1.0], [2.0]]), _rows([[1.0], [2.0]]))
    memory.fail = True
    with pytest.raises(RuntimeError):
        cache.append(_rows([[3.0] * 70, [4.0] * 70]), _rows([[3.0] * 70, [4.0] * 70]))
    memory.fail = False
    assert cache.lengths == (1, 1)
    cache.append(_rows([[5.0], [6.0]]), _rows([[5.0], [6.0]]))
    assert _held(cache, 0) == [1.0, 5.0] and _held(cache, 1) == [2.0, 6.0]


def test_refusals(memory):
    for sizes in ((0, 2, 32, 10), (1, 2, 32, 0)):
        with pytest.raises(ValueError, match="positive"):
            nn.PagedKVCache(*sizes, device="hip")
    for kw in ({"page_size": 0}, {"num_pages": 0}):
        with pytest.raises(ValueError, match="positive"):
            nn.PagedKVCache(1, 2, 32, 10, device="hip", **kw)
    with pytest.raises(NotImplementedError, match="head dims"):
        nn.PagedKVCache(1, 2, 48, 10, device="hip")
    with pytest.raises(RuntimeError, match="hip devices"):
        nn.PagedKVCache(1, 2, 32, 10, device="cpu")
    with pytest.raises(TypeError):
        nn.PagedKVCache(1, 2, 32, 10, device="hip", dtype="float64")
    cache = nn.PagedKVCache(2, 2, 32, 100, device="hip", num_pages=3)
    x = lambda *s, **kw: ts.Tensor(torch.zeros(s), device="hip", **kw)  # noqa: E731
    good = x(2, 2, 1, 32)
    for k, v, what in ((x(2, 2, 1, 64), good, "key shape"), (x(2, 3, 1, 32), good, "key shape"),
                       (x(2, 2, 32), good, "key shape"), (good, x(2, 2, 2, 32), "value shape"),
                       (x(2, 2, 0, 32), x(2, 2, 0, 32), "capacity 100"), (x(2, 2, 101, 32), x(2, 2, 101, 32), "capacity"),
                       (ts.Tensor(np.zeros((2, 2, 1, 32), np.float32)), good, "same device")):
        with pytest.raises(ValueError, match=what):
            cache.append(k, v)
    with pytest.raises(RuntimeError, match="inference-only"):
        cache.append(x(2, 2, 1, 32, requires_grad=True), good)
    for base in (0.0, -1.0, float("inf")):
        with pytest.raises(ValueError, match="RoPE"):
            cache.append(good, good, rotary_base=base)
    with pytest.raises(ValueError, match="exhausted: 4 pages needed, 3 free"):
        cache.append(x(2, 2, 65, 32), x(2, 2, 65, 32))
    assert cache.lengths == (0, 0) and cache.pages_in_use == 0 and (cache._core.host < 0).all()
    cache.append(good, good)
    for length in (2, -1, [1], [1, 2], 1.0, [[1, 1]]):
        with pytest.raises(ValueError, match="truncate"):
            cache.truncate(length)
    for index in ([0], [0, 2], [0, -1], [0.0, 1.0]):
        with pytest.raises(ValueError, match="beam ind"):
            cache.reorder(index)
    for index in ([], [0, 0], [2], [-1], [0.5], 0):
        with pytest.raises(ValueError, match="row"):
            cache.rows(index)
    for index in ([2], [-1], [0.5], [[0]]):
        with pytest.raises(ValueError, match="row ind"):
            cache.free(index)
    for last in (0, 2, -1):
        with pytest.raises(ValueError, match="last positions"):
            cache.get(last=last)
    for call in (cache.compact, cache.copy):
        with pytest.raises(ValueError, match="2 pages are in use"):
            call(1)
    q = x(2, 4, 1, 32)
    for query, what, error in ((x(2, 4, 32), "expects", ValueError), (x(1, 4, 1, 32), "query shape", ValueError),
                               (x(2, 4, 1, 64), "query shape", ValueError), (x(2, 3, 1, 32), "grouped", ValueError),
                               (x(2, 4, 0, 32), "grouped", ValueError),
                               (ts.Tensor(torch.zeros(2, 4, 1, 32).half(), device="hip"), "dtype", TypeError),
                               (x(2, 4, 1, 32, requires_grad=True), "inference-only", RuntimeError)):
        with pytest.raises(error, match=what):
            nn.paged_attention(query, cache)
    for kw in ({"scale": float("nan")}, {"rotary_base": 0.0}):
        with pytest.raises(ValueError):
            nn.paged_attention(q, cache, **kw)
    attention = nn.MultiHeadAttention(64, 2, device="hip").eval()
    with pytest.raises(ValueError, match="4 bits"):
        attention.new_cache(2, 100, quantized=True, paged=True)
    ragged = attention.new_cache(2, 100, paged=True)
    ragged.rows([1]).append(x(1, 2, 3, 32), x(1, 2, 3, 32))
    with ts.no_grad(), pytest.raises(ValueError, match="one length"):
        attention(x(2, 1, 64), cache=ragged, attn_mask=ts.Tensor(torch.ones(2, 1, 1, 4, dtype=torch.bool), device="hip"))


def test_the_prompt_rule():
    """Both sides of each measured crossing, runs of equal rows counted once."""
    lens = lambda *n: np.array(n, np.int32)  # noqa: E731
    for rows, heads, dim, wide, n, codes in (
            (128, 8, 128, False, lens(8000), True), (512, 8, 128, False, lens(8000), False),
            (1024, 8, 128, False, lens(500), True), (2048, 8, 128, False, lens(2000), False),
            (1024, 8, 128, True, lens(8000), True), (1024, 2, 64, False, lens(8000), True),
            (256, 8, 128, False, lens(8000, 8000, 8000), False), (256, 8, 128, False, lens(8000, 7000, 7500), True),
            (4096, 8, 128, True, lens(32000), True), (32, 4, 64, False, lens(0), True),
            (1 << 18, 1, 64, True, lens(300), True), ((1 << 18) + 1, 1, 64, True, lens(300), False),
            (1 << 17, 8, 128, True, lens(16384), True), (1 << 17, 8, 128, True, lens(32769), False)):
        assert P._reads_codes(rows, heads, dim, wide, n) is codes, (rows, heads, dim, wide, n)
    assert P._runs(lens(3, 3, 5, 3)) == [2, 3, 4] and P._runs(lens(7)) == [1]


def test_outgrown_rope_tables_stay():
    """A captured append reads the table that it was captured with."""
    A = importlib.import_module("tensorsmith_hip.nn.attention")
    make = lambda n: A.rope_tables(77.0, 32, torch.float32, torch.device("cpu"), n)  # noqa: E731
    kept = [(weakref.ref(t), t.clone()) for t in make(10)]
    long = make(3000)
    gc.collect()
    assert all(ref() is not None and torch.equal(ref(), old) for ref, old in kept)
    assert all(torch.equal(t[:len(old)], old) for t, (_, old) in zip(long, kept)) and make(20) is long


# -- the C entry points: every refusal comes before a launch --------------------------


def _ints(*x):
    return (ctypes.c_int32 * len(x))(*x)


def _desc(**kw):
    d = _lib.Pages4()
    d.pool, d.num_pages, d.heads, d.page_size, d.dim = 0x10000, 8, 2, 64, 128
    d.table, d.table_rows, d.table_stride = 0x20000, 4, 3
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def _rows_view(d=128, heads=2, steps=1, **kw):
    v = _lib.View()
    v.data = kw.get("data", 0x40000)
    for i, s in enumerate(kw.get("stride", (heads * steps * d, steps * d, d, 1))):
        v.stride[i] = s
    return v


OK_CALL = {"desc": {}, "dtype": _lib.F16, "rows": (0, 1), "lens": (5, 6), "steps": 1, "view": {}, "cos": None, "sin": None}
BAD = [
    ({"dtype": _lib.F64}, _lib.ERR_INVALID, "dtype"),
    ({"rows": (0, 4)}, _lib.ERR_INVALID, "table row 4"),
    ({"rows": (-1, 0)}, _lib.ERR_INVALID, "table row -1"),
    ({"lens": (5, 193)}, _lib.ERR_INVALID, "193 positions"),
    ({"lens": (-1, 0)}, _lib.ERR_INVALID, "-1 positions"),
    ({"steps": 0}, _lib.ERR_INVALID, "positive"),
    ({"desc": {"num_pages": 0}}, _lib.ERR_INVALID, "positive"),
    ({"desc": {"pool": None}}, _lib.ERR_INVALID, "NULL"),
    ({"desc": {"table": None}}, _lib.ERR_INVALID, "NULL"),
    ({"desc": {"pool": 0x10008}}, _lib.ERR_UNSUPPORTED, "16-byte"),
    ({"desc": {"dim": 96}}, _lib.ERR_UNSUPPORTED, "head dims"),
    ({"desc": {"page_size": 48}}, _lib.ERR_UNSUPPORTED, "pages of"),
    ({"desc": {"page_size": 8192}}, _lib.ERR_UNSUPPORTED, "pages of"),
    ({"view": {"data": None}}, _lib.ERR_INVALID, "NULL"),
    ({"view": {"data": 0x40008}}, _lib.ERR_UNSUPPORTED, "16-byte"),
    ({"view": {"stride": (256, 128, 4, 1)}}, _lib.ERR_UNSUPPORTED, "16-byte"),
    ({"view": {"stride": (256, 128, 128, 2)}}, _lib.ERR_INVALID, "innermost"),
    ({"cos": 0x1000}, _lib.ERR_INVALID, "both"),
    ({"cos": 0x1000, "sin": 0x2008}, _lib.ERR_UNSUPPORTED, "16-byte"),
]


def _calls(**kw):
    c = {**OK_CALL, **kw}
    lib, d, v = _lib.load(), _desc(**c["desc"]), _rows_view(**c["view"])
    rows, lens = _ints(*c["rows"]), _ints(*c["lens"])
    n = len(c["rows"])
    append = lambda: lib.tsattn_pages4_append(d, c["dtype"], n, c["steps"], v, v, rows, lens, c["cos"], c["sin"], None)  # noqa: E731
    attend = lambda: lib.tsattn_pages4_attend(d, c["dtype"], n, 4, c["steps"], 0.1, 1, v, v, rows, lens, c["cos"],  # noqa: E731
                                              c["sin"], None, 0, None)
    read = lambda: lib.tsattn_pages4_read(d, c["dtype"], n, c["steps"], v, v, rows, lens, _ints(*[0] * n), None)  # noqa: E731
    return append, attend, read


@pytest.mark.parametrize("change,status,what", BAD, ids=lambda x: str(x) if isinstance(x, dict) else None)
def test_c_calls_refuse(change, status, what):
    calls = _calls(**change)
    for call in calls[:2] if "cos" in change else calls:
        assert call() == status and what in _lib.last_error()


def test_c_appends_attention_and_reads_refuse():
    lib = _lib.load()
    append, _, _ = _calls(rows=(1, 1))
    assert append() == _lib.ERR_INVALID and "different" in _lib.last_error()
    append, _, _ = _calls(lens=(5, 190), steps=3)
    assert append() == _lib.ERR_INVALID and "exceed" in _lib.last_error()
    d, v, rows, lens = _desc(), _rows_view(), _ints(0), _ints(150)
    call = lambda heads=4, scale=0.1, steps=1: lib.tsattn_pages4_attend(  # noqa: E731
        d, _lib.F16, 1, heads, steps, scale, 1, v, v, rows, lens, None, None, None, 0, None)
    assert call(heads=3) == _lib.ERR_INVALID and "divisible" in _lib.last_error()
    assert call(heads=0) == _lib.ERR_INVALID
    assert call(scale=float("inf")) == _lib.ERR_INVALID and "finite" in _lib.last_error()
    assert call(steps=1 << 20) == _lib.ERR_UNSUPPORTED
    d.table_stride, lens = 300, _ints(19000)
    need = lib.tsattn_pages4_attend_workspace(d, _lib.F16, 1, 4, 1, lens)
    assert need > 0
    assert lib.tsattn_pages4_attend(d, _lib.F16, 1, 4, 1, 0.1, 1, v, v, rows, lens, None, None, 0x1000, need - 1,
                                    None) == _lib.ERR_INVALID and "too small" in _lib.last_error()
    assert lib.tsattn_pages4_read(d, _lib.F16, 1, 1, v, v, rows, lens, _ints(-1), None) == _lib.ERR_INVALID
    for lens in ((-1,), (1 << 28,)):
        assert lib.tsattn_pages4_attend_workspace(d, _lib.F16, 1, 4, 1, _ints(*lens)) == 0
    d.heads, d.table_stride = 4096, 1 << 21  # (more tiles, heads and sides than a launch numbers)
    for call in (lambda: lib.tsattn_pages4_append(d, _lib.F16, 1, 1 << 26, v, v, rows, _ints(0), None, None, None),
                 lambda: lib.tsattn_pages4_read(d, _lib.F16, 1, 1 << 26, v, v, rows, _ints(0), _ints(0), None)):
        assert call() == _lib.ERR_UNSUPPORTED and "too many" in _lib.last_error()
    assert lib.tsattn_pages4_page_bytes(8, 64, 128) == 8 * 2 * 36 * 128
    assert [lib.tsattn_pages4_page_bytes(*s) for s in ((8, 64, 96), (8, 33, 64), (0, 64, 64), (8, 16, 64))] == [0] * 4


def test_c_tables_refuse():
    lib = _lib.load()
    arrays = {name: np.zeros(n, np.int32) for name, n in (("table", 6), ("lengths", 3), ("refs", 4), ("stack", 4),
                                                          ("shown", 6), ("changed", 6), ("dirty", 2))}
    h = _lib.Pages4Host()
    h.rows, h.columns, h.page_size, h.pages, h.free = 3, 2, 32, 4, 4
    arrays["table"][:], arrays["shown"][:], arrays["stack"][:] = -1, -1, (3, 2, 1, 0)
    for name, x in arrays.items():
        setattr(h, name, x.ctypes.data)
    src, dst, copies = _ints(*[0] * 4), _ints(*[0] * 4), _ints(0)
    grow = lambda rows, steps, src=src: lib.tsattn_pages4_grow(h, len(rows), _ints(*rows), steps, src, dst, copies)  # noqa: E731
    for bad in (grow([3], 1), grow([-1], 1), grow([0, 0], 1), grow([], 1), grow([0], 0), grow([0], 65),
                grow([0], 1, None), lib.tsattn_pages4_grow(None, 1, _ints(0), 1, src, dst, copies),
                grow([0, 1, 2], 64)):
        assert bad == _lib.ERR_INVALID
    assert "6 pages needed, 4 free" in _lib.last_error() and h.free == 4 and (arrays["table"] < 0).all()
    for stack in ((3, 2, 1, 4), (3, 2, -1, 0)):  # (a free page that the pool does not have)
        arrays["stack"][:] = stack
        assert grow([0, 1], 1) == _lib.ERR_INVALID and h.free == 4 and (arrays["table"] < 0).all()
    arrays["stack"][:] = (3, 2, 1, 0)
    for length in (-1, 65):  # (past the table)
        arrays["lengths"][1] = length
        assert grow([1], 1) == lib.tsattn_pages4_compact(h, src, dst, copies) == _lib.ERR_INVALID
    arrays["lengths"][1] = 0
    assert grow([0, 2], 33) == 0 and h.free == 0 and h.n_changed == 4
    arrays["lengths"][:] = (33, 0, 33)
    cut = lambda rows, lens: lib.tsattn_pages4_cut(h, len(rows), _ints(*rows), _ints(*lens))  # noqa: E731
    assert [cut([0], [34]), cut([0], [-1]), cut([1], [1]), cut([0, 0], [1, 1])] == [_lib.ERR_INVALID] * 4
    order = lambda index: lib.tsattn_pages4_reorder(h, len(index), _ints(0, 1, 2), _ints(*index))  # noqa: E731
    assert [order([0, 1, 3]), order([-1, 0, 0])] == [_lib.ERR_INVALID] * 2
    held, after = arrays["table"].copy(), arrays["refs"].copy()
    for page in (-1, 4):  # (a held page that the pool does not have)
        arrays["table"][1] = page
        for bad in (grow([0], 1), cut([0], [0]), order([1, 0, 2]), lib.tsattn_pages4_compact(h, src, dst, copies)):
            assert bad == _lib.ERR_INVALID and f"page {page} of 4" in _lib.last_error()
        assert lib.tsattn_pages4_clone(h, 3, _ints(0, 1, 2), h, src, dst, copies) == _lib.ERR_INVALID
    arrays["table"][:] = held
    assert (arrays["refs"] == after).all() and h.free == 0 and arrays["lengths"].tolist() == [33, 0, 33]
    to = _lib.Pages4Host()
    for name, _ in _lib.Pages4Host._fields_:
        setattr(to, name, getattr(h, name))
    clone = lambda n: lib.tsattn_pages4_clone(h, n, _ints(0, 1, 2), to, src, dst, copies)  # noqa: E731
    assert clone(2) == _lib.ERR_INVALID and "columns" in _lib.last_error()
    to.pages = 3
    assert clone(3) == _lib.ERR_INVALID and "4 pages are in use" in _lib.last_error()
    to.table = None
    assert clone(3) == _lib.ERR_INVALID
    copy = lambda src, dst, to=0x10000, pages=8, size=1024, table=0x1000: lib.tsattn_pages4_apply(  # noqa: E731
        h, table, 0x10000, 8, to, pages, size, len(src), _ints(*src), _ints(*dst), None)
    for bad in (copy([0, 1], [2, 2]), copy([0, 1], [1, 2]), copy([8], [0]), copy([0], [8]), copy([-1], [0]),
                copy([0], [3], to=0x50000, pages=3), copy([3], [3]), copy([], [], table=None), copy([0], [1], to=None),
                lib.tsattn_pages4_apply(h, 0x1000, 0x10000, 8, 0x10000, 8, 1024, -1, None, None, None)):
        assert bad == _lib.ERR_INVALID
    assert copy([0], [1], size=1000) == copy([0], [1], to=0x50008) == _lib.ERR_UNSUPPORTED and h.n_changed == 4
    assert lib.tsattn_pages4_compact(h, src, None, copies) == _lib.ERR_INVALID
    h.free = 1  # (every page is held)
    assert lib.tsattn_pages4_compact(h, src, dst, copies) == _lib.ERR_INVALID and "4 pages are held" in _lib.last_error()
    h.free = 5
    assert lib.tsattn_pages4_compact(h, src, dst, copies) == _lib.ERR_INVALID
