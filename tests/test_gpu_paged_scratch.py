"""Paged attention whose partial sums pass 4 GiB, taken in parts (needs an MI355X):
sequences of very unequal lengths, and one sequence of very many rows, against float64.
"""

from __future__ import annotations

import importlib
import math
from unittest.mock import patch

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("no GPU", allow_module_level=True)

from test_gpu_paged import BF16, F32, check, draw, reference, say, seeded, stored, wrap  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402

P = importlib.import_module("tensorsmith_hip.nn.paged")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_long_sequence_beside_short_ones(dtype):
    say("paged scratch, unequal lengths", dtype)
    gen, hkv, d, steps, b = seeded(21), 8, 256, 512, 64
    lens = [100 + 7 * i for i in range(b)]
    lens[41] = 131_100
    cache = nn.PagedKVCache(b, hkv, d, max(lens), device="hip", dtype=dtype, page_size=256,
                            num_pages=sum(-(-n // 256) for n in lens))
    parts = []
    for i, n in enumerate(lens):
        k, v = (draw(gen, 1, hkv, n, d, dtype=dtype) for _ in range(2))
        cache.rows([i]).append(wrap(k), wrap(v))
        parts.append((k, v))
    q = draw(gen, b, hkv, steps, d, dtype=dtype)
    with patch.object(P, "_reads_codes", return_value=True):
        got = nn.paged_attention(wrap(q), cache)._data
    for i in (0, 31, 32, 41, 63):
        heads, (k, v) = slice(0, None, 7), parts[i]
        t = 3 if i == 41 else steps  # (of the long one the last queries)
        want, tol = reference(q[i:i + 1, heads, -t:], stored(k[:, heads]), stored(v[:, heads]), [lens[i]], True,
                              1 / math.sqrt(d), False)
        check(got[i:i + 1, heads, -t:], want, tol, dtype)


def test_one_sequence_of_very_many_rows():
    say("paged scratch, many rows")
    gen, hkv, rep, d, steps, n = seeded(22), 8, 32, 256, 8192, 8300
    k, v = (draw(gen, 1, hkv, n, d, dtype=BF16) for _ in range(2))
    cache = nn.PagedKVCache(1, hkv, d, n, device="hip", dtype=BF16)
    cache.append(wrap(k), wrap(v))
    q = draw(gen, 1, hkv * rep, steps, d, dtype=BF16)
    got = nn.paged_attention(wrap(q), cache)._data
    sk, sv = stored(k), stored(v)
    for h in (0, 7):
        for r in (0, 15, 16, 31):
            head = h * rep + r
            for t in (0, 4095, 4096, 8191):  # (a query alone: what it sees are the positions up to its own)
                seen = n - steps + t + 1
                want, tol = reference(q[:, head:head + 1, t:t + 1], sk[:, h:h + 1, :seen], sv[:, h:h + 1, :seen], [seen],
                                      True, 1 / math.sqrt(d), False)
                check(got[:, head:head + 1, t:t + 1], want, tol, BF16)
