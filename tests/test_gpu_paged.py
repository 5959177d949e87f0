"""The paged 4-bit cache against its definition in float64 (needs an MI355X): what an
append keeps, attention over it, pages that rows share, and a model's cached steps.

Tolerances.  Stored values are exact.  Attention: a score's fp32 sum of D products is
off by at most (D + 8) 2^-24 of the sum of their magnitudes, which moves each
probability by that much of itself, twice over (the numerator's and the
denominator's); the value products enter within 2^-17 (fp32: 2^-24) and their n
terms sum in fp32: (n / 16 + 16) 2^-24, sixteen at a time or fewer.  All relative to the
largest value of the row's head, and the result's own rounding on top.  The prompt path
rounds each probability to 16 bits once more.
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

import tensorsmith_hip as ts  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402

P = importlib.import_module("tensorsmith_hip.nn.paged")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HALF = {F16: 2.0**-11, BF16: 2.0**-8, F32: 2.0**-24}
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
BORDERS = (LEVELS[1:] + LEVELS[:-1]) / 2


def say(*x):
    print(*x, flush=True)


def wrap(x):
    return ts.Tensor(x, device="hip")


def draw(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def seeded(n):
    return torch.Generator(device="cuda").manual_seed(n)


def stored(x):
    """The format's values of rows x, in float64 on the host."""
    dtype, g = x.dtype, x.double().cpu().reshape(*x.shape[:-1], -1, 32)
    most = 10752.0 if dtype == F16 else 1.3125 * 2.0**125
    m = g.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp((m / 6).float().double())
    s = torch.ldexp(torch.round(mantissa * 64) / 64, exponent).clamp(2.0**-27, most)
    y = (g / s).abs()
    low, high = torch.bucketize(y, BORDERS), torch.bucketize(y, BORDERS, right=True)
    value = LEVELS[torch.where(low % 2 == 0, low, high).clamp(0, 7)] * s
    value = torch.where(g < 0, -value, value)
    return torch.where(torch.isfinite(g).all(-1, keepdim=True), value, math.nan).reshape(x.shape)


def same(got, want, dtype):
    """Equal as the dtype holds it (a NaN anywhere both have one)."""
    want = want.to(dtype).double()
    return torch.equal(torch.nan_to_num(got.double().cpu(), nan=7e77), torch.nan_to_num(want, nan=7e77))


def held(cache):
    return [x._data for x in cache.get()]


# -- append and read --------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,h,steps,page", [(32, 3, (1, 1, 62, 1), 64), (64, 2, (33, 31, 5), 32), (128, 2, (77, 1, 50), 64),
                                            (256, 1, (9, 32, 23), 128)])
def test_appends_keep_the_nearest_codes(d, h, steps, page, dtype):
    say("append", d, h, steps, page, dtype)
    gen, b = seeded(d), 3
    cache = nn.PagedKVCache(b, h, d, 200, device="hip", dtype=dtype, page_size=page)
    x = [[draw(gen, b, h, n, d, dtype=dtype, scale=2.0 ** (3 * i - 4)) for n in steps] for i in range(2)]
    for k, v in zip(*x):
        cache.append(wrap(k), wrap(v))
    for got, rows in zip(held(cache), x):
        assert same(got, stored(torch.cat(rows, 2)), dtype)
    for last in (1, sum(steps) - 1, sum(steps)):
        for got, rows in zip(cache.get(last=last), x):
            assert same(got._data, stored(torch.cat(rows, 2)[:, :, -last:]), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_appends_round_ties_edges_and_extremes(dtype):
    """Ties at every border, on scales of all mantissas; zeros, the smallest and the largest groups."""
    say("append edges", dtype)
    rows = []
    for i in range(32, 64):  # scales of 6 bits: 32/32 .. 63/32
        s = i / 32 * 2.0 ** (i % 5 - 2)
        ties = torch.cat((BORDERS, -BORDERS, torch.nextafter(BORDERS.float(), torch.tensor(9.0)).double(),
                          torch.nextafter(BORDERS.float(), torch.tensor(0.0)).double(), torch.tensor([6.0, -6.0, 0.0, 1.0])))
        rows.append(ties * s)
    tiny = torch.finfo(dtype).tiny
    top = torch.finfo(dtype).max
    for m in (0.0, 6 * 2.0**-27, 2.0**-26, tiny, torch.finfo(dtype).smallest_normal, top, top / 1.01, top / 2, 1.0,
              63.4 / 64 * 6, 6 * (1 + 1 / 64), 6 * (1 + 3 / 64)):  # (scales' own ties)
        rows.append(torch.linspace(-1, 1, 32, dtype=torch.float64) * m)
    x = torch.stack(rows).to(dtype).cuda()[None, None]
    cache = nn.PagedKVCache(1, 1, 32, x.shape[2], device="hip", dtype=dtype)
    cache.append(wrap(x), wrap(-x))
    k, v = held(cache)
    assert same(k, stored(x), dtype) and same(v, stored(-x), dtype)
    assert torch.isfinite(k).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_groups_that_are_not_finite_read_as_nan(dtype):
    """And only they; attention over positions that do not see them stays finite."""
    say("append not finite", dtype)
    gen = seeded(5)
    k, v = (draw(gen, 2, 2, 70, 64, dtype=dtype) for _ in range(2))
    k[0, 0, 65, 3], k[1, 1, 69, 40], v[0, 1, 66, 0], v[1, 0, 64, 63] = math.inf, math.nan, -math.inf, math.nan
    cache = nn.PagedKVCache(2, 2, 64, 100, device="hip", dtype=dtype)
    cache.append(wrap(k), wrap(v))
    got = held(cache)
    for x, y in zip(got, (k, v)):
        assert same(x, stored(y), dtype) and torch.isnan(x).sum() == 64
    q = draw(gen, 2, 2, 10, 64, dtype=dtype)
    out = nn.paged_attention(wrap(q), cache)._data  # positions 60 .. 69: the first four see none of them
    assert torch.isfinite(out[:, :, :4]).all() and torch.isnan(out[0, 0, 5:]).all() and torch.isnan(out[1, 1, 9]).all()
    assert torch.isnan(out[0, 1, 6:, :32]).all() and torch.isfinite(out[0, 1, 6:, 32:]).all()
    cache.truncate(64)
    assert torch.isfinite(nn.paged_attention(wrap(q[:, :, :1].contiguous()), cache)._data).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_of_any_strides(dtype):
    say("append strides", dtype)
    gen = seeded(8)
    base = draw(gen, 2, 40, 3, 64, dtype=dtype)
    for x in (base.permute(0, 2, 1, 3), draw(gen, 2, 3, 40, 65, dtype=dtype)[..., 1:],
              draw(gen, 2, 3, 64, 40, dtype=dtype).transpose(2, 3), draw(gen, 1, 1, 40, 64, dtype=dtype).expand(2, 3, 40, 64)):
        cache = nn.PagedKVCache(2, 3, 64, 50, device="hip", dtype=dtype)
        cache.append(wrap(x), wrap(x))
        assert all(same(y, stored(x), dtype) for y in held(cache))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_keys_rotate_at_their_rows_positions(d, dtype):
    say("append rotary", d, dtype)
    gen, lens = seeded(d), (0, 31, 100)
    cache = nn.PagedKVCache(3, 2, d, 200, device="hip", dtype=dtype)
    past = draw(gen, 3, 2, 100, d, dtype=dtype)
    cache.append(wrap(past), wrap(past))
    cache.truncate(lens)
    k, v = (draw(gen, 3, 2, 35, d, dtype=dtype) for _ in range(2))
    cache.append(wrap(k), wrap(v), rotary_base=10000.0)
    got = cache.get(last=35)
    for i, n in enumerate(lens):
        turned = nn.rotary_embedding(wrap(k[i:i + 1]), n)._data
        assert same(got[0]._data[i:i + 1], stored(turned), dtype) and same(got[1]._data[i:i + 1], stored(v[i:i + 1]), dtype)
        if n:
            assert same(held(cache.rows([i]))[0][:, :, :n], stored(past[i:i + 1, :, :n]), dtype)


# -- attention --------------------------------------------------------------------


def reference(q, k, v, lens, causal, scale, prompt):
    """Attention in float64 of q over stored values k, v, and how far a result may be off."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(*q.shape[:3], 1, dtype=torch.float64)
    rep, t, d = q.shape[1] // k.shape[1], q.shape[2], q.shape[3]
    eps = 2.0**-24
    for b, n in enumerate(lens):
        if n == 0:
            continue
        for h in range(q.shape[1]):
            kk, vv, qq = k[b, h // rep, :n], v[b, h // rep, :n], q[b, h].double().cpu()
            x = qq @ kk.t() * scale
            seen = torch.arange(n)[None] <= (torch.arange(t) + n - t)[:, None] if causal else torch.ones(t, n, dtype=torch.bool)
            x = x.masked_fill(~seen, -math.inf)
            p = torch.softmax(x, -1).nan_to_num(0.0)
            out[b, h] = p @ vv
            far = (qq.abs() @ kk.abs().t()).amax(-1, keepdim=True) * abs(scale)
            off = 2 * (d + 8) * eps * far + (n / 16 + 16) * eps + (2.0**-24 if q.dtype == F32 else 2.0**-17)
            tol[b, h] = (off + (HALF[q.dtype] if prompt else 0)) * vv.abs().max()
    return out, tol


def check(got, want, tol, dtype):
    err = (got.double().cpu() - want).abs() - HALF[dtype] * want.abs()
    assert (err <= tol + 1e-30).all(), ((err / (tol + 1e-30)).max().item(), tol.max().item())


CASES = [
    # heads, KV heads, steps, lengths, dim, page, dtype, causal
    (8, 8, 1, (1, 33), 64, 64, F16, True),
    (4, 4, 1, (31, 32, 0), 32, 32, F32, True),
    (8, 2, 1, (257, 64, 700), 128, 64, BF16, True),
    (6, 2, 1, (65, 1), 128, 32, F32, True),
    (2, 2, 3, (2, 128, 300, 0), 128, 128, F16, True),   # more queries than positions: the first see nothing
    (16, 2, 1, (1000, 513), 64, 64, BF16, True),
    (16, 1, 1, (40, 999), 32, 64, F16, True),
    (24, 1, 1, (70,), 128, 64, F16, True),              # three workgroups of rows
    (7, 1, 5, (333, 90), 64, 32, BF16, True),
    (4, 2, 1, (300, 1), 256, 64, BF16, True),
    (4, 2, 2, (97,), 256, 64, F32, True),
    (3, 3, 4, (64, 65), 256, 32, F16, False),
    (8, 4, 2, (3000, 10), 128, 64, BF16, True),         # several splits, a row that ends in the first
    (8, 4, 1, (5000, 4097, 1), 64, 256, F32, True),
    (4, 1, 9, (128, 8), 128, 64, F16, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).split(".")[-1].replace(" ", "") for x in c))
def test_attention_matches_float64(case):
    say("paged attention", case)
    heads, hkv, steps, lens, d, page, dtype, causal = case
    gen, b = seeded(heads + d + steps), len(lens)
    cache = nn.PagedKVCache(b, hkv, d, max(lens) + 9, device="hip", dtype=dtype, page_size=page)
    k, v = (draw(gen, b, hkv, max(lens), d, dtype=dtype) for _ in range(2))
    for i in range(0, max(lens), 500):  # (rows' pages lie among each other's)
        cache.append(wrap(k[:, :, i:i + 500]), wrap(v[:, :, i:i + 500]))
    cache.truncate(lens)
    q = draw(gen, b, heads, steps, d, dtype=dtype)
    want, tol = reference(q, stored(k), stored(v), lens, causal, 1 / math.sqrt(d), False)
    got = nn.paged_attention(wrap(q), cache, is_causal=causal)._data
    check(got, want, tol, dtype)
    assert torch.equal(got, nn.paged_attention(wrap(q), cache, is_causal=causal)._data)
    strided = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(got, nn.paged_attention(wrap(strided), cache, is_causal=causal)._data)
    off = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(got, nn.paged_attention(wrap(off), cache, is_causal=causal)._data)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,hkv,rep,steps,keys,d", [
    (16, 8, 4, 25, 40, 32), (24, 2, 4, 25, 500, 32), (1, 8, 4, 16, 4000, 32), (24, 1, 1, 1, 4000, 32),
    (8, 8, 4, 25, 40, 64), (24, 1, 4, 25, 500, 64), (1, 8, 4, 16, 4000, 64), (1, 1, 8, 8, 2500, 64),
    (4, 8, 4, 25, 40, 128), (24, 2, 4, 25, 300, 128), (1, 4, 8, 8, 1500, 128), (1, 4, 4, 16, 2500, 128),
    (1, 1, 1, 1, 200, 32), (1, 1, 1, 1, 2500, 32), (1, 1, 1, 1, 200, 64), (1, 1, 1, 1, 1500, 64),
    (1, 1, 1, 1, 200, 128), (1, 1, 1, 1, 1000, 128), (1, 1, 1, 1, 200, 256), (1, 1, 4, 25, 1500, 256),
])
def test_workgroups_of_every_make(batch, hkv, rep, steps, keys, d, dtype):
    """Shapes over which the plan takes one and two column blocks, four and eight waves, one split
    and several, for every head dim that has them; over the codes, whatever the rows' number."""
    say("paged workgroups", batch, hkv, rep, steps, keys, d, dtype)
    gen = seeded(keys + d)
    cache = nn.PagedKVCache(batch, hkv, d, keys, device="hip", dtype=dtype)
    k, v = (draw(gen, batch, hkv, keys, d, dtype=dtype) for _ in range(2))
    cache.append(wrap(k), wrap(v))
    lens = [keys - i % 3 * (keys // 7) for i in range(batch)]
    cache.truncate(lens)
    q = draw(gen, batch, hkv * rep, steps, d, dtype=dtype)
    want, tol = reference(q, stored(k), stored(v), lens, True, 1 / math.sqrt(d), False)
    with patch.object(P, "_reads_codes", return_value=True):
        check(nn.paged_attention(wrap(q), cache)._data, want, tol, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,rep", [(32, 1), (64, 4), (128, 1), (128, 8), (256, 8)])
def test_what_is_not_seen_does_not_count(d, rep, dtype):
    """NaN in later positions of the chunk, in cut ones and in pages never written: rows that do not
    see them are as they are without."""
    say("paged unseen NaN", d, rep, dtype)
    gen, steps, n = seeded(d + rep), 37, 150
    k, v = (draw(gen, 1, 2, n, d, dtype=dtype) for _ in range(2))
    q = draw(gen, 1, 2 * rep, steps, d, dtype=dtype)
    outs = []
    for bad in (False, True):
        kk, vv = k.clone(), v.clone()
        cache = nn.PagedKVCache(1, 2, d, 256, device="hip", dtype=dtype)
        if bad:
            kk[:, :, n - 5:], vv[:, :, n - 9] = math.nan, math.nan  # seen by the last 5, by the last 9 queries
            cache._core.pool.fill_(0xFF)                            # (codes of 6, scales of NaN)
            x = torch.full((1, 2, 256, d), math.nan, dtype=dtype, device="cuda")
            cache.append(wrap(x), wrap(x))
            cache.truncate(0)
        cache.append(wrap(kk), wrap(vv))
        with patch.object(P, "_reads_codes", return_value=True):
            outs.append(nn.paged_attention(wrap(q), cache)._data)
    assert torch.equal(outs[0][:, :, :-9], outs[1][:, :, :-9])
    assert torch.isfinite(outs[0]).all() and torch.isnan(outs[1][:, :, -9:]).all()


@pytest.mark.parametrize("dtype,d", [(BF16, 32), (F32, 64)])
def test_rows_of_hundreds_of_thousands(dtype, d):
    """More splits than the second kernel has loads in flight, beside a row of one position."""
    say("paged long rows", dtype, d)
    gen, n = seeded(d), 300_001
    cache = nn.PagedKVCache(2, 1, d, n, device="hip", dtype=dtype, page_size=4096, num_pages=75)
    k, v = (draw(gen, 1, 1, n, d, dtype=dtype) for _ in range(2))
    cache.rows([0]).append(wrap(k), wrap(v))
    cache.rows([1]).append(wrap(k[:, :, :1]), wrap(v[:, :, :1]))
    assert cache.pages_in_use == 75
    q = draw(gen, 2, 2, 1, d, dtype=dtype, scale=3.0)
    sk, sv = (stored(x).expand(2, -1, -1, -1) for x in (k, v))
    want, tol = reference(q, sk, sv, (n, 1), True, 1 / math.sqrt(d), False)
    check(nn.paged_attention(wrap(q), cache)._data, want, tol, dtype)
    assert same(cache.rows([0]).get(last=5000)[0]._data, sk[:1, :, -5000:], dtype)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_any_scale(scale, dtype):
    say("paged attention scale", scale, dtype)
    gen = seeded(3)
    k, v = (draw(gen, 2, 2, 90, 64, dtype=dtype) for _ in range(2))
    cache = nn.PagedKVCache(2, 2, 64, 90, device="hip", dtype=dtype)
    cache.append(wrap(k), wrap(v))
    q = draw(gen, 2, 4, 1, 64, dtype=dtype)
    want, tol = reference(q, stored(k), stored(v), (90, 90), True, scale, False)
    check(nn.paged_attention(wrap(q), cache, scale=scale)._data, want, tol, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,heads,hkv,steps,lens", [(64, 4, 2, 70, (70, 70)), (128, 2, 2, 150, (333, 333)),
                                                    (32, 8, 2, 40, (41, 90, 90, 40)), (128, 8, 1, 33, (50, 700)),
                                                    (128, 8, 1, 33, (20, 100)), (256, 2, 1, 100, (130, 250))])
def test_prompts_match_float64(d, heads, hkv, steps, lens, dtype):
    """Chunks of prompts: rows of one length, of several, and with fewer positions than queries."""
    say("paged prompt", d, heads, hkv, steps, lens, dtype)
    gen, b = seeded(d + steps), len(lens)
    k, v = (draw(gen, b, hkv, max(lens), d, dtype=dtype) for _ in range(2))
    cache = nn.PagedKVCache(b, hkv, d, max(lens), device="hip", dtype=dtype)
    cache.append(wrap(k), wrap(v))
    cache.truncate(lens)
    q = draw(gen, b, heads, steps, d, dtype=dtype)
    for causal in (True, False):
        for codes in (True, False):  # from the codes, and from values dequantised once
            want, tol = reference(q, stored(k), stored(v), lens, causal, 1 / math.sqrt(d), not codes)
            with patch.object(P, "_reads_codes", lambda *a: codes):
                check(nn.paged_attention(wrap(q), cache, is_causal=causal)._data, want, tol, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,heads,steps", [(32, 2, 3), (64, 4, 1), (128, 2, 2), (256, 2, 1), (64, 4, 80)])
def test_queries_rotate_at_their_positions(d, heads, steps, dtype):
    say("paged rotary", d, heads, steps, dtype)
    gen, lens = seeded(d), (100, 81)
    cache = nn.PagedKVCache(2, 2, d, 100, device="hip", dtype=dtype)
    k, v = (draw(gen, 2, 2, 100, d, dtype=dtype) for _ in range(2))
    cache.append(wrap(k), wrap(v), rotary_base=500.0)
    cache.truncate(lens)
    q = draw(gen, 2, heads, steps, d, dtype=dtype)
    turned = torch.cat([nn.rotary_embedding(wrap(q[i:i + 1]), n - steps, base=500.0)._data for i, n in enumerate(lens)])
    for codes in (True, False):
        with patch.object(P, "_reads_codes", lambda *a: codes):
            got = nn.paged_attention(wrap(q), cache, rotary_base=500.0)._data
            assert torch.equal(got, nn.paged_attention(wrap(turned), cache)._data)


def test_many_sequences_and_far_pages():
    """More rows than a launch takes, and pages past 4 GiB of the pool."""
    gen, b, h, d = seeded(1), 300, 8, 128
    say("paged, many rows, far pages")
    cache = nn.PagedKVCache(b, h, d, 64, device="hip", dtype=BF16, num_pages=65000)
    assert cache._core.pool.numel() > 2**32
    core = cache._core
    core.stack[:] = core.stack[::-1].copy()  # the last pages are given out first
    k, v = (draw(gen, b, h, 40, d, dtype=BF16) for _ in range(2))
    cache.append(wrap(k), wrap(v))
    assert int(core.host[core.host >= 0].min()) * core.page_bytes > 2**32
    lens = [1 + (7 * i) % 40 for i in range(b)]
    cache.truncate(lens)
    ks, vs = stored(k), stored(v)
    got = held(cache)
    for i in (0, 255, 256, 299):
        assert same(got[0][i, :, :lens[i]], ks[i, :, :lens[i]], BF16) and not got[1][i, :, lens[i]:].any()
    q = draw(gen, b, 8, 1, d, dtype=BF16)
    out = nn.paged_attention(wrap(q), cache)._data
    index = [0, 1, 255, 256, 299]
    want, tol = reference(q[index], ks[index], vs[index], [lens[i] for i in index], True, 1 / math.sqrt(d), False)
    check(out[index], want, tol, BF16)
    assert cache.compact() == b
    assert torch.equal(out, nn.paged_attention(wrap(q), cache)._data)


# -- pages ------------------------------------------------------------------------


def test_shared_pages_are_copied_for_the_row_that_appends():
    say("paged forks")
    gen, h, d = seeded(2), 4, 128
    prompt, new, more = (draw(gen, n, h, s, d, dtype=F16) for n, s in ((1, 100), (5, 1), (5, 70)))
    cache = nn.PagedKVCache(5, h, d, 300, device="hip", dtype=F16)
    cache.rows([2]).append(wrap(prompt), wrap(-prompt))
    cache.reorder([2] * 5)
    assert cache.pages_in_use == 2
    cache.append(wrap(new), wrap(-new))
    want = torch.cat((prompt.expand(5, -1, -1, -1), new), 2)
    k, v = held(cache)
    assert same(k, stored(want), F16) and same(v, stored(-want), F16)
    cache.reorder([4, 4, 0, 1, 1])  # beams: rows taken over again
    cache.append(wrap(more), wrap(-more))
    want = torch.cat((want[[4, 4, 0, 1, 1]], more), 2)
    assert same(held(cache)[0], stored(want), F16)
    snapshot = cache.copy()
    cache.free([0, 3])
    cache.rows([3, 0]).append(wrap(new[:2]), wrap(new[:2]))
    assert cache.lengths == (1, 171, 171, 1, 171)
    before = held(cache)
    assert cache.compact() == cache.pages_in_use and all(torch.equal(x, y) for x, y in zip(before, held(cache)))
    cache.compact(cache.pages_in_use + 5)
    assert all(torch.equal(x, y) for x, y in zip(before, held(cache)))
    assert same(before[0][:1, :, :1], stored(new[1:2]), F16) and same(before[0][1:3], stored(want[1:3]), F16)
    assert same(held(snapshot)[1], stored(-want), F16)
    q = draw(gen, 5, 8, 1, d, dtype=F16)
    want64, tol = reference(q, stored(want), stored(-want), [171] * 5, True, 1 / math.sqrt(d), False)
    check(nn.paged_attention(wrap(q), snapshot)._data, want64, tol, F16)


def test_pages_of_every_size_copy_whole():
    say("page copies")
    gen = seeded(4)
    for h, d, page, dtype in ((1, 32, 32, F32), (3, 64, 128, F16), (8, 128, 512, BF16), (5, 256, 64, F16)):
        cache = nn.PagedKVCache(2, h, d, 700, device="hip", dtype=dtype, page_size=page)
        x = draw(gen, 2, h, 650, d, dtype=dtype)
        cache.append(wrap(x), wrap(-x))
        other = cache.copy(num_pages=cache.pages_in_use)
        cache.reset()
        cache.append(wrap(-x), wrap(x))
        k, v = held(other)
        assert same(k, stored(x), dtype) and same(v, stored(-x), dtype) and same(held(cache)[0], stored(-x), dtype)


# -- streams, graphs ---------------------------------------------------------------


def test_on_another_stream_and_captured():
    """A captured append and attention replay the positions they were captured at, eager work between."""
    say("paged capture")
    gen = seeded(6)
    cache = nn.PagedKVCache(3, 2, 64, 3000, device="hip", dtype=BF16)
    k, v = (draw(gen, 3, 2, 2000, 64, dtype=BF16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(wrap(k), wrap(v))
        cache.truncate([2000, 70, 1500])
        new = [draw(gen, 3, 2, 1, 64, dtype=BF16) for _ in range(3)]
        q = draw(gen, 3, 4, 1, 64, dtype=BF16)
        kt, vt, qt = new[0].clone(), new[0].clone(), q.clone()
        cache.append(wrap(kt), wrap(vt), rotary_base=100.0)  # (its pages are there now)
        cache.truncate([2000, 70, 1500])
        cache.append(wrap(kt), wrap(vt), rotary_base=100.0)
        nn.paged_attention(wrap(qt), cache, rotary_base=100.0)
        lens = [n - 1 for n in cache.lengths]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    full = nn.PagedKVCache(3, 2, 64, 128, device="hip", dtype=BF16)
    full.append(*(wrap(x[:, :, :64].contiguous()) for x in (k, v)))
    shared = full.copy()
    shared.truncate(40)
    shared.reorder([0, 0, 1])
    assert all(torch.equal(x, y[[0, 0, 1], :, :40]) for x, y in zip(held(shared), held(full)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: full.append(wrap(kt), wrap(vt)), full.copy, full.compact, lambda: shared.append(wrap(kt), wrap(vt))):
            with pytest.raises(RuntimeError, match="cannot change while a graph"):
                call()
        core = cache._core
        core.lengths -= 1  # (the captured append writes where the eager one did)
        cache.append(wrap(kt), wrap(vt), rotary_base=100.0)
        out = nn.paged_attention(wrap(qt), cache, rotary_base=100.0)._data
    for i in range(4):
        kt.copy_(new[i % 3]), vt.copy_(new[(i + 1) % 3]), qt.copy_(q * (i + 1))
        graph.replay()
        got, keys = out.clone(), [x._data.clone() for x in cache.get(last=1)]
        torch.cuda.synchronize()
        cache.truncate(lens)
        cache.append(wrap(new[i % 3]), wrap(new[(i + 1) % 3]), rotary_base=100.0)
        assert torch.equal(got, nn.paged_attention(wrap((q * (i + 1))), cache, rotary_base=100.0)._data), i
        assert all(torch.equal(x, y._data) for x, y in zip(keys, cache.get(last=1)))
    assert full.lengths == (64, 64, 64) and full.pages_in_use == 3  # the refused call left nothing
    assert all(torch.equal(x, y[[0, 0, 1], :, :40]) for x, y in zip(held(shared), held(full)))
    full.append(wrap(kt), wrap(vt))
    assert same(held(full)[0][:, :, 64:], stored(kt), BF16) and same(held(full)[1][:, :, :64], stored(v[:, :, :64]), BF16)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_a_captured_rotation_outlives_its_table(dtype):
    """The tables of angles grow for longer rows; a captured call goes on reading its own."""
    say("paged capture, longer tables", dtype)
    gen, base = seeded(61), 41.0 if dtype == F32 else 43.0  # (no other test's tables)
    cache = nn.PagedKVCache(2, 2, 64, 200, device="hip", dtype=dtype)
    first = [draw(gen, 2, 2, 70, 64, dtype=dtype) for _ in range(2)]
    new, q = draw(gen, 2, 2, 1, 64, dtype=dtype), draw(gen, 2, 4, 1, 64, dtype=dtype)
    cache.append(*map(wrap, first), rotary_base=base)
    cache.append(wrap(new), wrap(new), rotary_base=base)
    want = nn.paged_attention(wrap(q), cache, rotary_base=base)._data
    cache.truncate(70)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nn.paged_attention(wrap(q), cache, rotary_base=base)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        cache.append(wrap(new), wrap(new), rotary_base=base)
        out = nn.paged_attention(wrap(q), cache, rotary_base=base)._data
    for n in (700, 3000, 9000):
        far = nn.PagedKVCache(1, 2, 64, n, device="hip", dtype=dtype)
        x = draw(gen, 1, 2, n, 64, dtype=dtype)
        far.append(wrap(x), wrap(x), rotary_base=base)
        junk = [torch.full((m, 32), 9.0, dtype=dtype, device="cuda") for m in (256, 256, 700, 700)]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        del junk, far


# -- layers and models -------------------------------------------------------------


def _model(dtype, heads=4, kv_heads=2, dim=128):
    ts.seed(3)
    model = nn.TransformerLM(nn.TransformerConfig(vocab_size=97, dim=dim, num_heads=heads, num_kv_heads=kv_heads,
                                                  num_layers=2, max_seq_len=300), device="hip").eval()
    for p in model.parameters():
        p._data = p._data.to(dtype)
    return model


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_the_attention_layer_steps_over_it(dtype):
    """Rows at positions of their own, against the layer's parts and attention in float64."""
    say("paged layer", dtype)
    ts.seed(1)
    layer = nn.MultiHeadAttention(256, 4, num_kv_heads=2, device="hip").eval()
    for p in layer.parameters():
        p._data = p._data.to(dtype)
    cache = layer.new_cache(2, 200, dtype=dtype, paged=True)
    gen = seeded(1)
    x, y = draw(gen, 2, 90, 256, dtype=dtype), draw(gen, 2, 1, 256, dtype=dtype)
    with ts.no_grad():
        layer(wrap(x), cache=cache)
        cache.truncate([90, 41])
        out = layer(wrap(y), cache=cache)._data
        heads = lambda proj, z, n: proj(wrap(z)).reshape(z.shape[0], z.shape[1], n, 64).permute(0, 2, 1, 3)  # noqa: E731
        # what the cache holds is what the layer's projections give, rotated and stored
        k, v = (c._data for c in cache.get())
        for i, n in enumerate((90, 41)):
            z = torch.cat((x[i:i + 1, :n], y[i:i + 1]), 1)
            last = nn.rotary_embedding(heads(layer.k_proj, y, 2), n)._data[i:i + 1]
            assert same(k[i:i + 1, :, n:n + 1], stored(last), dtype)
            first = nn.rotary_embedding(heads(layer.k_proj, x, 2), 0)._data[i:i + 1, :, :n]
            assert same(k[i:i + 1, :, :n], stored(first), dtype) and z.shape[1] == n + 1
        q = heads(layer.q_proj, y, 4)
        q = torch.cat([nn.rotary_embedding(q, n)._data[i:i + 1] for i, n in enumerate((90, 41))])
        want, tol = reference(q, k.double().cpu(), v.double().cpu(), (91, 42), True, 1 / 8, False)
        w = layer.out_proj.weight._data.double().cpu()
        flat = lambda z: z.permute(0, 2, 1, 3).reshape(2, 1, 256)  # noqa: E731
        # the attended rows round to the dtype, then a product of 256 terms does
        wide = flat((tol + HALF[dtype] * want.abs()).expand(want.shape)) @ w.abs().t()
        wide = wide + 2 * 256 * 2.0**-24 * (flat(want).abs() @ w.abs().t())
        check(out, flat(want) @ w.t(), wide, dtype)


def test_a_mask_takes_the_values_read_back():
    say("paged layer, mask")
    ts.seed(2)
    layer = nn.MultiHeadAttention(128, 2, device="hip").eval()
    cache, plain = layer.new_cache(2, 64, paged=True), layer.new_cache(2, 64, paged=True)
    gen = seeded(2)
    x, y = draw(gen, 2, 20, 128), draw(gen, 2, 1, 128)
    with ts.no_grad():
        for c in (cache, plain):
            layer(wrap(x), cache=c)
        mask = torch.ones(2, 1, 1, 21, dtype=torch.bool, device="cuda")
        a = layer(wrap(y), cache=cache, attn_mask=wrap(mask))._data
        b = layer(wrap(y), cache=plain)._data
        # two orders of fp32 sums of the same values: 64 + 21 + 128 terms, scores of a few
        assert (a - b).abs().max() <= 64 * 2.0**-24 * b.abs().max() * 4


@pytest.mark.parametrize("dtype", [F32, F16])
def test_models_generate_and_serve_rows_of_their_own(dtype):
    """A whole batch's steps equal the same rows' alone; generation runs on it; a failed forward rolls back."""
    say("paged model", dtype)
    model = _model(dtype)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 97, (1, n), generator=gen).cuda() for n in (40, 7, 133)]
    nxt = torch.randint(0, 97, (3, 1), generator=gen).cuda()
    with ts.no_grad():
        together = model.new_cache(3, 200, paged=True)
        alone = [model.new_cache(1, 200, paged=True) for _ in prompts]
        for i, p in enumerate(prompts):
            model(wrap(p), caches=[c.rows([i]) for c in together])
            model(wrap(p), caches=alone[i])
        for a, b in zip(together, zip(*alone)):
            assert a.lengths == (40, 7, 133)
            for i, c in enumerate(b):
                assert all(torch.equal(x._data, y._data) for x, y in zip(a.rows([i]).get(), c.get()))
        logits = model(wrap(nxt), caches=together)._data
        for i in range(3):
            one = model(wrap(nxt[i:i + 1]), caches=alone[i])._data
            # (products of three rows and of one may sum in another order: their roundings
            # move stored codes, a step of 1/6 .. 1/3 of a group's largest, here and there)
            rel = (logits[i:i + 1] - one).float().norm() / one.float().norm()
            assert rel <= 0.05, rel
        assert {c.lengths for c in together} == {(41, 8, 134)}
        out = model.generate(wrap(prompts[0]), 12, temperature=0, paged_cache=True)._data
        assert out.shape == (1, 52) and torch.equal(out[:, :40], prompts[0])
        broken = model.blocks[1].ffn
        model.blocks[1].ffn = None
        with pytest.raises(Exception):
            model(wrap(nxt), caches=together)
        model.blocks[1].ffn = broken
        assert {c.lengths for c in together} == {(41, 8, 134)}
        with pytest.raises(ValueError, match="same sequence position"):
            together[0].truncate([40, 8, 134])
            model(wrap(nxt), caches=together)
