"""Codes over the whole range of scales (needs an MI355X): ties and their neighbours on
scales of every mantissa, up to the largest that a cache has, against float64."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("no GPU", allow_module_level=True)

from test_gpu_paged import BF16, BORDERS, F16, F32, held, same, say, stored, wrap  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_ties_on_every_scale(dtype):
    say("codes", dtype)
    rows, low, high = [], -27, 13 if dtype == F16 else 125
    near = torch.cat((BORDERS, -BORDERS)).to(dtype)
    ties = torch.cat((near, torch.nextafter(near, torch.tensor(9.0, dtype=dtype)),
                      torch.tensor([6.0, 0.5, 0.0, -6.0], dtype=dtype)))  # (a group's largest is 6 scales)
    for e in range(low, high + 1):
        for m in range(32, 64):
            s = m / 32 * 2.0 ** e
            if s <= (10752.0 if dtype == F16 else 1.3125 * 2.0 ** 125) and 6 * s >= 64 * torch.finfo(dtype).tiny:
                rows.append(ties.double() * s)
    x = torch.stack(rows).to(dtype).cuda()
    n = x.shape[0] // 2 * 2
    x = x[:n].view(1, 1, n // 2, 64)
    cache = nn.PagedKVCache(1, 1, 64, n // 2, device="hip", dtype=dtype)
    cache.append(wrap(x), wrap(-x))
    k, v = held(cache)
    assert same(k, stored(x), dtype) and same(v, stored(-x), dtype)
    assert torch.isfinite(k).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_groups_of_any_values(dtype):
    say("codes, large", dtype)
    gen = torch.Generator(device="cuda").manual_seed(31)
    x = torch.randn((1, 1, 4000, 256), generator=gen, device="cuda")
    size = torch.randint(60, 126, (1, 1, 4000, 1), generator=gen, device="cuda").float()
    x = (x.clamp(-3.9, 3.9) * torch.exp2(size)).to(dtype)
    x[..., ::9] = x[..., ::9] * 2.0 ** -100  # (values of no size beside them)
    cache = nn.PagedKVCache(1, 1, 256, 4000, device="hip", dtype=dtype)
    cache.append(wrap(x), wrap(-x))
    assert all(same(y, stored(z), dtype) for y, z in zip(held(cache), (x, -x)))
