"""Paged attention in every way that it is run (needs an MI355X): against float64, with
queries rotated at their rows' positions, and with NaN wherever a row does not see.

Tolerances as in ``test_gpu_paged``.
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

from paged_makes import SHAPES, key, lengths, plan  # noqa: E402
from test_gpu_paged import BF16, F16, F32, check, draw, reference, say, seeded, stored, wrap  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402

P = importlib.import_module("tensorsmith_hip.nn.paged")


@pytest.mark.parametrize("make", SHAPES, ids=lambda x: "-".join(map(str, x)))
def test_every_kernel(make):
    say("paged make", make, SHAPES[make])
    (name, d, *_), shape = make, SHAPES[make]
    dtype, (b, hkv, rep, steps, keys, _), lens = {"F32": F32, "F16": F16, "BF16": BF16}[name], shape, lengths(shape)
    assert key(name, d, plan(name, d, shape)) == make
    gen = seeded(keys + d)
    cache = nn.PagedKVCache(b, hkv, d, keys + 70, device="hip", dtype=dtype)
    k, v = (draw(gen, b, hkv, keys, d, dtype=dtype) for _ in range(2))
    cache.append(wrap(k), wrap(v), rotary_base=None)
    cache.truncate(lens)
    q = draw(gen, b, hkv * rep, steps, d, dtype=dtype)
    with patch.object(P, "_reads_codes", return_value=True):
        got = nn.paged_attention(wrap(q), cache)._data
        seen = sorted({0, b // 2, b - 1})
        heads = sorted({0, hkv - 1})
        for i in seen:
            for h in heads:
                rows = slice(h * rep, (h + 1) * rep)
                sk, sv = (stored(x[i:i + 1, h:h + 1]) for x in (k, v))
                want, tol = reference(q[i:i + 1, rows], sk, sv, [lens[i]], True, 1 / math.sqrt(d), False)
                check(got[i:i + 1, rows], want, tol, dtype)

        # rotated queries: as the same ones rotated before
        turned = torch.cat([nn.rotary_embedding(wrap(q[i:i + 1]), n - steps, base=300.0)._data for i, n in enumerate(lens)])
        assert torch.equal(nn.paged_attention(wrap(q), cache, rotary_base=300.0)._data,
                           nn.paged_attention(wrap(turned), cache)._data)

        # NaN in every row's last position, in cut positions and in pages never written
        junk = torch.full((b, hkv, keys + 70, d), math.nan, dtype=dtype, device="cuda")
        cache.truncate(0)
        cache._core.pool.fill_(0xFF)
        cache.append(wrap(junk), wrap(junk))
        cache.truncate(0)
        bad = [x.clone() for x in (k, v)]
        for i, n in enumerate(lens):
            for x in bad:
                x[i, :, n - 1:] = math.nan
        cache.append(*map(wrap, bad))
        cache.truncate(lens)
        out = nn.paged_attention(wrap(q), cache)._data
    assert torch.equal(out[:, :, :-1], got[:, :, :-1]) and torch.isnan(out[:, :, -1]).all()
