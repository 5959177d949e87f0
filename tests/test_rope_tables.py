"""The RoPE tables that launches share: made once, whichever threads ask for them."""

from __future__ import annotations

import importlib
import threading
import time

import numpy as np
import pytest

torch = pytest.importorskip("torch")

A = importlib.import_module("tensorsmith_hip.nn.attention")


def test_threads_get_one_table(monkeypatch):
    """A launch of either thread may still read what it was given: nothing replaces it unkept."""
    cos = np.cos
    monkeypatch.setattr(A.np, "cos", lambda x: (time.sleep(0.05), cos(x))[1])
    start, got = threading.Barrier(2), [None, None]

    def ask(i, length):
        start.wait()
        got[i] = A.rope_tables(79.0, 32, torch.float32, torch.device("cpu"), length)

    for length in (10, 5000):
        workers = [threading.Thread(target=ask, args=(i, length)) for i in range(2)]
        for w in workers:
            w.start()
        for w in workers:
            w.join()
        assert got[0][0] is got[1][0] and got[0][1] is got[1][1]
        assert got[0][0].shape[0] >= length
