"""Views of one paged cache stepped by several threads: what one call changes in the page
tables and what it brings to the device belong together.

The kernels stand in as in ``test_paged_host``; a page update lets the other threads run
before its work, as a library call that holds no interpreter lock does.
"""

from __future__ import annotations

import threading
import time

import pytest

torch = pytest.importorskip("torch")

from test_paged_host import Memory, _rows, _sound, memory  # noqa: E402, F401
from tensorsmith_hip import nn  # noqa: E402


class Yielding(Memory):
    def tsattn_pages4_apply(self, *a):
        time.sleep(2e-4)
        return super().tsattn_pages4_apply(*a)

    def tsattn_pages4_append(self, *a):
        time.sleep(1e-4)
        return super().tsattn_pages4_append(*a)


@pytest.mark.parametrize("threads", [2, 4])
def test_threads_fork_append_and_free_rows_of_their_own(memory, threads):  # noqa: F811
    memory.__class__ = Yielding
    cache = nn.PagedKVCache(2 * threads, 2, 32, 300, device="hip", page_size=32)
    want, errors = [[] for _ in range(2 * threads)], []
    start = threading.Barrier(threads)

    def work(i):
        try:
            view, mine, tag = cache.rows([2 * i, 2 * i + 1]), [[], []], 1000.0 * i
            start.wait()
            for step in range(12):
                new = [[tag + k for k in range(5)], [tag + 5 + k for k in range(5)]]
                tag += 10
                view.append(_rows(new), _rows(new))
                mine = [x + y for x, y in zip(mine, new)]
                if step % 3 == 1:
                    view.reorder([1, 1])
                    mine = [list(mine[1]), list(mine[1])]
                if step % 5 == 4:
                    view.truncate([len(mine[0]) - 3, 0])
                    mine = [mine[0][:-3], []]
            want[2 * i], want[2 * i + 1] = mine
        except BaseException as error:  # noqa: BLE001
            errors.append(error)

    workers = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for w in workers:
        w.start()
    for w in workers:
        w.join()
    assert not errors
    _sound(cache, want)
