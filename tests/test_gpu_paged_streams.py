"""The paged cache on several streams of one device (needs an MI355X): pages that are
given back and taken again while the stream that reads them is behind.
"""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("no GPU", allow_module_level=True)

from test_gpu_paged import BF16, F16, draw, held, same, say, seeded, stored, wrap  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402


def _behind():
    """Some ten milliseconds of work on the current stream."""
    x = torch.ones(8192, 8192, dtype=BF16, device="cuda")
    for _ in range(12):
        y = x @ x
    return y


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_freed_rows_pages_wait_for_their_last_reader(dtype):
    say("paged streams", dtype)
    gen, b, h, d, n = seeded(11), 4, 2, 128, 640
    cache = nn.PagedKVCache(b, h, d, n, device="hip", dtype=dtype, num_pages=2 * n // 64)
    k, v = (draw(gen, 2, h, n, d, dtype=dtype) for _ in range(2))
    cache.rows([0, 1]).append(wrap(k), wrap(v))
    q = draw(gen, 2, 4, 1, d, dtype=dtype)
    want = nn.paged_attention(wrap(q), cache.rows([0, 1]))._data.clone()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        _behind()
        got = nn.paged_attention(wrap(q), cache.rows([0, 1]))._data
        keys = cache.rows([0, 1]).get()[0]._data
    with torch.cuda.stream(second):
        cache.free([0, 1])
        cache.rows([3, 2]).append(wrap(-v), wrap(-k))  # (every page of the pool is taken again)
        new = held(cache.rows([3, 2]))
    torch.cuda.synchronize()
    assert torch.equal(got, want) and same(keys, stored(k), dtype)
    assert same(new[0], stored(-v), dtype) and same(new[1], stored(-k), dtype)


def test_a_cache_made_on_one_stream_and_used_on_another():
    """Its pool lies where a buffer was whose last writer is still queued."""
    say("paged streams, new cache")
    gen = seeded(12)
    x = draw(gen, 1, 8, 4096, 128, dtype=BF16)
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        cache = nn.PagedKVCache(1, 8, 128, 4096, device="hip", dtype=BF16)
        shape = cache._core.pool.shape
        del cache
        buffer = torch.empty(shape, dtype=torch.uint8, device="cuda")
        _behind()
        buffer.fill_(0xFF)
        del buffer
        cache = nn.PagedKVCache(1, 8, 128, 4096, device="hip", dtype=BF16)
    with torch.cuda.stream(second):
        cache.append(wrap(x), wrap(x))
        got = held(cache)
    torch.cuda.synchronize()
    assert all(same(y, stored(x), BF16) for y in got)
