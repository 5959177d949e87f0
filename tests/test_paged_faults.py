"""Page updates that fail: rows of the paged cache keep their positions, and what the
device lacks is sent by the next call.

The kernels stand in as in ``test_paged_host`` (a tag a position in CPU memory), with a
page update that fails before its work or amid it, or is interrupted before or after.
"""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_host import Memory, _at, _held, _ints, _rows, _sound, memory  # noqa: E402, F401
from tensorsmith_hip import _lib, nn  # noqa: E402


class Stop(BaseException):
    """An interrupt."""


class Failing(Memory):
    """``when``: where the next page update that has something to do fails."""

    when = None

    def tsattn_pages4_apply(self, host, table, source, sn, target, tn, page_bytes, n, src, dst, stream):
        when, self.when = self.when, None
        if when == "before":
            return _lib.ERR_HIP
        if when == "amid":
            first = _at(src, n, np.int32)[:n // 2], _at(dst, n, np.int32)[:n // 2]
            old, new = (_at(x, m * page_bytes, np.uint8).reshape(m, -1) for x, m in ((source, sn), (target, tn)))
            new[first[1]] = old[first[0]]
            return _lib.ERR_HIP
        if when == "interrupt":
            raise Stop
        rc = super().tsattn_pages4_apply(host, table, source, sn, target, tn, page_bytes, n, src, dst, stream)
        if when == "after":
            raise Stop
        return rc


@pytest.fixture
def failing(memory):  # noqa: F811
    memory.__class__ = Failing
    return memory


WHEN = ("before", "amid", "interrupt", "after")


@pytest.mark.parametrize("when", WHEN)
def test_a_row_that_shares_its_page_keeps_it(failing, when):
    """Two rows of [1, 2]; the copy for one of them fails; the next append finds both as they were."""
    cache = nn.PagedKVCache(2, 2, 32, 100, device="hip", num_pages=4)
    cache.rows([0]).append(_rows([[1.0, 2.0]]), _rows([[1.0, 2.0]]))
    cache.reorder([0, 0])
    failing.when = when
    with pytest.raises((RuntimeError, Stop)):
        cache.append(_rows([[3.0] * 70, [4.0] * 70]), _rows([[3.0] * 70, [4.0] * 70]))
    assert cache.lengths == (2, 2) and cache.pages_in_use <= 2
    cache.append(_rows([[7.0], [8.0]]), _rows([[7.0], [8.0]]))
    _sound(cache, [[1.0, 2.0, 7.0], [1.0, 2.0, 8.0]])


@pytest.mark.parametrize("when", WHEN)
@pytest.mark.parametrize("then", ["append", "reorder", "free", "truncate", "reset", "compact", "copy", "get", "attend"])
def test_any_call_after_it_brings_the_device_up_to_date_first(failing, when, then):
    failing.tsattn_pages4_read = failing.tsattn_pages4_attend = lambda *a: 0  # noqa: E731
    failing.tsattn_pages4_attend_workspace = lambda *a: 0
    cache = nn.PagedKVCache(3, 2, 32, 100, device="hip", page_size=32)
    cache.append(_rows([[1.0] * 40, [2.0] * 40, [3.0] * 40]), _rows([[0.0] * 40] * 3))
    cache.free([0])
    failing.when = when
    with pytest.raises((RuntimeError, Stop)):
        cache.compact()  # (row 2's pages move to the front)
    want = [[], [2.0] * 40, [3.0] * 40]
    other = None
    if then == "append":
        cache.append(_rows([[4.0] * 33] * 3), _rows([[0.0] * 33] * 3))
        want = [x + [4.0] * 33 for x in want]
    elif then == "reorder":
        cache.reorder([2, 1, 1])
        want = [want[2], want[1], want[1]]
    elif then == "free":
        cache.free([1])
        want[1] = []
        cache.rows([0]).append(_rows([[5.0] * 70]), _rows([[5.0] * 70]))
        want[0] = [5.0] * 70
    elif then == "truncate":
        cache.truncate([0, 3, 40])
        want[1] = want[1][:3]
    elif then == "reset":
        cache.rows([1]).reset()
        want[1] = []
    elif then == "compact":
        cache.compact(9)
    elif then == "copy":
        other = cache.copy()
    elif then == "get":
        cache.get()
    else:
        nn.paged_attention(_rows([[1.0]] * 3), cache)
    _sound(cache, want)
    if other is not None:
        _sound(other, want)


@pytest.mark.parametrize("seed", range(12))
def test_rows_keep_their_positions_through_failures(failing, seed):
    rng = random.Random(seed)
    b, page = rng.choice([2, 3, 5]), rng.choice([32, 64])
    full = b * -(-300 // page)
    cache = nn.PagedKVCache(b, 2, 32, 300, device="hip", page_size=page, num_pages=rng.choice([full, full * 2 // 3]))
    want, tag, failed = [[] for _ in range(b)], 1.0, 0
    for _ in range(150):
        failing.when = rng.choice([None, *WHEN])
        failing.fail = rng.random() < 0.1  # the append's own launch
        what = rng.choice(["append"] * 5 + ["reorder", "cut", "free", "compact", "resize", "copy"])
        index = rng.sample(range(b), rng.randint(1, b))
        try:
            if what == "append":
                n = rng.choice([1, 1, 2, rng.randint(1, 70)])
                if max(len(want[i]) for i in index) + n > 300:
                    continue
                new = [[tag + i * n + j for j in range(n)] for i in range(len(index))]
                tag += len(index) * n
                cache.rows(index).append(_rows(new), _rows(new))
                for i, x in zip(index, new):
                    want[i] = want[i] + x
            elif what == "reorder":
                index = [rng.randrange(b) for _ in range(b)]
                moved = [list(want[i]) for i in index]
                pending = failing.when  # (an earlier call's update may be what fails)
                before = cache.lengths, cache._core.host.copy()
                try:
                    cache.reorder(index)
                except (RuntimeError, Stop):
                    assert pending
                    if cache.lengths == before[0] and (cache._core.host == before[1]).all():
                        moved = want
                    raise
                finally:
                    want = moved
            elif what == "cut":
                lens = [max(0, len(x) - rng.choice([0, 1, 40])) for x in want]
                cache.truncate(lens)
                want = [x[:n] for x, n in zip(want, lens)]
            elif what == "free":
                cache.free(index)
                want = [[] if i in index else x for i, x in enumerate(want)]
            elif what == "compact":
                cache.compact()
            elif what == "resize":
                cache.compact(max(1, cache.pages_in_use + rng.choice([0, 1, full])))
            else:
                other = cache.copy()
                _sound(other, want)
        except (RuntimeError, Stop):
            failed += 1
        except ValueError as error:
            assert "pool exhausted" in str(error)
        failing.when, failing.fail = None, False
        if rng.random() < 0.5:
            cache._core.ready()
            _sound(cache, want)
    cache._core.ready()
    _sound(cache, want)
    assert failed > 5


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launch has to fail: no device")
def test_c_updates_that_fail_are_still_to_be_sent():
    lib = _lib.load()
    arrays = {name: np.zeros(n, np.int32) for name, n in (("table", 4), ("lengths", 2), ("refs", 4), ("stack", 4),
                                                          ("shown", 4), ("changed", 4), ("dirty", 1))}
    h = _lib.Pages4Host()
    h.rows, h.columns, h.page_size, h.pages, h.free = 2, 2, 32, 4, 4
    arrays["table"][:], arrays["shown"][:], arrays["stack"][:] = -1, -1, (3, 2, 1, 0)
    for name, x in arrays.items():
        setattr(h, name, x.ctypes.data)
    src, dst, copies = _ints(*[0] * 4), _ints(*[0] * 4), _ints(0)
    assert lib.tsattn_pages4_grow(h, 2, _ints(0, 1), 33, src, dst, copies) == 0 and h.n_changed == 4
    memory = ctypes.create_string_buffer(64)
    for _ in range(2):
        assert lib.tsattn_pages4_apply(h, ctypes.addressof(memory), None, 0, None, 0, 0, 0, None, None, None) == _lib.ERR_HIP
        assert h.n_changed == 4 and (arrays["shown"] == -1).all() and (arrays["dirty"].view(np.uint8) == 1).all()
