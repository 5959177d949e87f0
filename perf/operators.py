"""Keys and values held in 4 bits, in pages: the append that quantises, the attention
that reads them, and copies and forks of pages.

The format, for each 32 channels of a row x: a scale s of 6 significant bits,
``s = round6(max|x| / 6)`` (the quotient in fp32) between 2^-27 and the largest whose
multiples the cache's dtype holds, and a code a channel: the nearest of 0, 0.5, 1, 1.5,
2, 3, 4, 6 to |x| / s, ties to the even code, with a sign.  Its value is the code's
level times s.

A case is a dict of plain values; ``kind`` says what one pass does:

* ``attend``: ``nn.paged_attention`` of new queries over a cache of rows of unequal
  lengths: one token a row, a few drafted ones, or a chunk of a prompt;
* ``append``: ``PagedKVCache.append`` of new keys (rotated at each row's own
  positions) and values, and the stored values of the new positions read back;
* ``fork``: rows take over a prompt's pages (``reorder``), append a token each, which
  copies the page that they share, and read their last positions back;
* ``copy``: ``PagedKVCache.copy``, and the copy's values.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAGE = 64
GROUP = 32
BITS = 4.5  # a channel: the code, and its share of a 16-bit scale


def _framework():
    path = os.path.join(os.getcwd(), "custom-ml-library_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tensorsmith_hip as ts

    return ts


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _attend(name, dtype, batch, heads, kv_heads, tokens, keys, dim, ragged):
    case = {"kind": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "tokens": tokens, "keys": keys, "dim": dim, "ragged": ragged}
    return {"name": name, **case} if name else case


def _append(name, dtype, batch, kv_heads, tokens, past, dim, ragged, rotary):
    case = {"kind": "append", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "tokens": tokens,
            "past": past, "dim": dim, "ragged": ragged, "rotary": rotary}
    return {"name": name, **case} if name else case


def _pages(name, kind, dtype, batch, kv_heads, keys, dim, ragged):
    case = {"kind": kind, "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "keys": keys, "dim": dim,
            "ragged": ragged}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one stream early in its answer: the smallest call, launches and host work count
        _attend("attend_f16_b1h8_k200", "f16", 1, 8, 2, 1, 200, 64, False),
        # the default model's heads (4 of 32 channels) and dtype, a small batch
        _attend("attend_f32_b16h4_k900_d32", "f32", 16, 4, 4, 1, 900, 32, True),
        # serving a batch through grouped-query heads, one new token a sequence
        _attend("attend_f16_b64h32kv8_k1025", "f16", 64, 32, 8, 1, 1025, 128, False),
        # long contexts of unequal length, as many KV heads as query heads
        _attend("attend_bf16_b64h32_k8192", "bf16", 64, 32, 32, 1, 8192, 128, True),
        # five drafted tokens a row to verify
        _attend("attend_bf16_b7h16kv4_t5_k4001", "bf16", 7, 16, 4, 5, 4001, 128, True),
        # one chunk of a long prompt over the cache of what came before
        _attend("attend_bf16_t500_k8192", "bf16", 1, 32, 8, 500, 8192, 128, False),
        # a decoding step's new rows, each at its own position
        _append("append_f16_b64kv8_t1", "f16", 64, 8, 1, 1025, 128, True, True),
        # prompts of a batch
        _append("append_bf16_b4kv8_t8192", "bf16", 4, 8, 8192, 0, 128, False, True),
        # drafted tokens in the default dtype, from odd positions
        _append("append_f32_b3h4_t77_d64", "f32", 3, 4, 77, 333, 64, True, True),
        # eight beams start from one prompt
        _pages("fork_f16_b8kv8_k1000", "fork", "f16", 8, 8, 1000, 128, False),
        # a snapshot of a batch's cache, its pages scattered over the pool
        _pages("copy_bf16_b16kv8_k4001", "copy", "bf16", 16, 8, 4001, 128, True),
        # and of one short conversation
        _pages("copy_f16_b1h8_k333_d64", "copy", "f16", 1, 8, 333, 64, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    dim = rng.choice([32, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    batch, keys, ragged = _log(rng, 1, 64), _log(rng, 1, 16000), rng.random() < 0.6
    pick = rng.random()
    most = 64 * 8 * 8192 * 128
    if pick < 0.55:
        rep = rng.choice([1, 2, 4, 7, 8])
        tokens = rng.choice([1, 1, 1, 2, 5, 9])
        if rng.random() < 0.25:
            tokens, batch = _log(rng, 10, 1000), min(batch, 3)
        keys = max(keys, tokens)
        while batch * kv_heads * keys * dim > most or batch * kv_heads * rep * tokens * keys > 4e8:
            if batch > 1:
                batch //= 2
            elif keys // 2 >= tokens:
                keys //= 2
            else:
                tokens //= 2
        return _attend(None, dtype, batch, kv_heads * rep, kv_heads, tokens, keys, dim, ragged)
    if pick < 0.8:
        tokens, past = rng.choice([1, 1, 3, _log(rng, 2, 6000)]), rng.choice([0, keys])
        while batch * kv_heads * max(past, tokens) * dim > 4 * 8 * 8192 * 128:
            batch, past = max(1, batch // 2), past // 2
        return _append(None, dtype, batch, kv_heads, tokens, past, dim, ragged and past > 0, rng.random() < 0.7)
    while batch * kv_heads * keys * dim > 16 * 8 * 4096 * 128:
        batch, keys = max(1, batch // 2), max(1, keys // 2)
    if pick < 0.9:
        return _pages(None, "fork", dtype, batch, kv_heads, keys, dim, False)
    return _pages(None, "copy", dtype, batch, kv_heads, keys, dim, ragged)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _lengths(case, seed):
    """Cached positions of every row: all of them, or spread over (n / 16, n] in an order of the seed's."""
    b, n = case["batch"], case["past" if case["kind"] == "append" else "keys"]
    if not case["ragged"] or n == 0:
        return [n] * b
    least = case.get("tokens", 1) if case["kind"] == "attend" else 1
    low = n // 16
    all_ = [max(least, low + int((n - low) * (i + 1) / b)) for i in range(b)]
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
    return [all_[i] for i in order]


def _rows(gen, case, tokens, spread):
    """Keys or values [B, H, tokens, D]; `spread`: how unequal the channels are (keys' are)."""
    d, dtype = case["dim"], TORCH[case["dtype"]]
    channels = torch.exp(spread * torch.randn(d, generator=gen, device=DEV)).to(dtype)
    x = torch.randn((case["batch"], case["kv_heads"], tokens, d), generator=gen, device=DEV, dtype=dtype)
    return x.mul_(channels)


def _inputs(case, seed):
    """What one pass works on, from the seed alone: cached rows, then the new ones."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lengths(case, seed)
    got = {"lens": lens}
    if max(lens):
        got["past"] = (_rows(gen, case, max(lens), 0.6), _rows(gen, case, max(lens), 0.2))
    if case["kind"] == "attend":
        shape = (case["batch"], case["heads"], case["tokens"], case["dim"])
        got["q"] = torch.randn(shape, generator=gen, device=DEV, dtype=TORCH[case["dtype"]])
    if case["kind"] in ("append", "fork"):
        tokens = case.get("tokens", 1)
        got["new"] = (_rows(gen, case, tokens, 0.6), _rows(gen, case, tokens, 0.2))
    return got


def _angles(case, positions):
    """cos and sin [positions, D / 2] of the rotary embedding, in the cache's dtype."""
    d = case["dim"]
    freqs = 10000.0 ** (-np.arange(0, d, 2, dtype=np.float32) / np.float32(d))
    at = np.arange(positions, dtype=np.float32)[:, None] * freqs[None, :]
    return [torch.from_numpy(np.ascontiguousarray(f(at))).to(DEV, TORCH[case["dtype"]]) for f in (np.cos, np.sin)]


def _capacity(case):
    n = case["past"] + case["tokens"] if case["kind"] == "append" else case["keys"] + 1
    return n + PAGE


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# half way between two levels, and whether it belongs to the upper one (the even code)
BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
LEAST = 2.0 ** -27
MOST = {torch.float16: 10752.0, torch.bfloat16: 1.3125 * 2.0 ** 125, torch.float32: 1.3125 * 2.0 ** 125}


def _quantise(x):
    """Rows [..., D] -> two codes a byte [..., D / 2] and scales [..., D / 32] (bf16 holds their 6 bits)."""
    a = x.float().unflatten(-1, (-1, GROUP))
    s = (a.abs().amax(-1).double() / 6.0).float()  # (fp32 by a number may multiply by its reciprocal)
    bits = s.view(torch.int32)
    bits = (bits + 0x1FFFF + ((bits >> 18) & 1)) & ~0x3FFFF  # to the nearest of 6 bits, ties to even
    s = bits.view(torch.float32).clamp(LEAST, MOST[x.dtype])[..., None]
    size = a.abs()
    code = (a < 0).to(torch.uint8) * 8
    for at, up in BORDERS:  # (a border's few bits times the scale's 6 are exact)
        code += (size >= at * s) if up else (size > at * s)
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, s[..., 0].to(torch.bfloat16)


def _dequantise(codes, scales):
    """The fp32 values of packed rows."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)[c.int()]
    return (level.unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _rotate(x, cos, sin):
    """Interleaved pairs by each position's angle; every product and sum rounds to x's dtype."""
    t = x.dtype
    r = lambda z: z.to(t).float()  # noqa: E731
    even, odd, c, s = x[..., 0::2].float(), x[..., 1::2].float(), cos.float(), sin.float()
    return torch.stack((r(r(even * c) - r(odd * s)), r(r(odd * c) + r(even * s))), -1).flatten(-2).to(t)


class _Pool:
    """Pages [n, H, PAGE, ...] of keys and values, and the page of every row's every 64 positions."""

    def __init__(self, batch, heads, dim, pages_a_row):
        n = batch * pages_a_row
        side = lambda: (torch.zeros((n, heads, PAGE, dim // 2), dtype=torch.uint8, device=DEV),  # noqa: E731
                        torch.zeros((n, heads, PAGE, dim // GROUP), dtype=torch.bfloat16, device=DEV))
        self.sides = (side(), side())
        self.table = torch.arange(n, device=DEV).view(pages_a_row, batch).t().contiguous()

    def write(self, rows, at):
        """Rows (keys, values) [B, H, T, D] at the positions `at` [B, T]."""
        page = torch.gather(self.table, 1, at // PAGE)
        for x, (codes, scales) in zip(rows, self.sides):
            c, s = _quantise(x)
            codes[page, :, at % PAGE], scales[page, :, at % PAGE] = c.transpose(1, 2), s.transpose(1, 2)

    def read(self, at):
        """The values of the positions `at` [B, T]: keys, values [B, H, T, D] in fp32."""
        page = torch.gather(self.table, 1, at // PAGE)
        return [_dequantise(c[page, :, at % PAGE], s[page, :, at % PAGE]).transpose(1, 2) for c, s in self.sides]


def _plain_attend(state):
    case, pool, q = state["case"], state["pool"], state["q"]
    b, h, t, d = q.shape
    n, lens = max(state["lens"]), state["lens_dev"]
    k, v = pool.read(torch.arange(n, device=DEV).expand(b, n))
    q = q.float().reshape(b, case["kv_heads"], -1, d)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(d))
    seen = torch.arange(n, device=DEV) <= (lens[:, None] - t + torch.arange(t, device=DEV))[..., None]
    x = x.view(b, h, t, n).masked_fill_(~seen[:, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, case["kv_heads"], -1, n), v.contiguous()).view(b, h, t, d)
    return (out / total).to(state["q"].dtype)


def _plain_append(state):
    case = state["case"]
    k, v = state["new"]
    t = case.get("tokens", 1)
    at = state["lens_dev"][:, None] + torch.arange(t, device=DEV)
    if case.get("rotary"):
        k = _rotate(k, state["cos"][at][:, None], state["sin"][at][:, None])
    state["pool"].write((k, v), at)
    return [x.to(k.dtype) for x in state["pool"].read(at)]


def _plain_fork(state):
    """Every row's pages become copies of row 0's (the shared ones are read where they are), then a token each."""
    case, pool, n = state["case"], state["pool"], state["lens"][0]
    b, full = case["batch"], n // PAGE
    pool.table[1:, :full] = pool.table[0, :full].clone()
    if n % PAGE:
        for side in pool.sides:
            for x in side:
                x[pool.table[1:, full]] = x[pool.table[0, full]].clone()
    state["lens_dev"] = torch.full((b,), n, device=DEV)
    _plain_append(state)
    last = min(n + 1, PAGE)
    at = torch.arange(n + 1 - last, n + 1, device=DEV).expand(b, last)
    return [x.to(TORCH[case["dtype"]]) for x in pool.read(at)]


def _plain_copy(state):
    case, pool, n = state["case"], state["pool"], max(state["lens"])
    table = pool.table[:, : -(-n // PAGE)]
    new = [[x[table.reshape(-1)] for x in side] for side in pool.sides]
    at = torch.arange(n, device=DEV).expand(case["batch"], n)
    live = (at < state["lens_dev"][:, None])[:, None, :, None]
    page = torch.arange(table.numel(), device=DEV).view(table.shape).gather(1, at // PAGE)
    values = [_dequantise(c[page, :, at % PAGE], s[page, :, at % PAGE]).transpose(1, 2) for c, s in new]
    return [torch.where(live, x, 0.0).to(TORCH[case["dtype"]]) for x in values]


# ---------------------------------------------------------------------------
# Entry points
# ---------------------------------------------------------------------------


def prepare(case, seed):
    got = _inputs(case, seed)
    state = {"case": case, "lens": got["lens"]}
    past, chunk = got.get("past"), 1000  # (filled as a server does: rows grow side by side)
    n = max(got["lens"])
    if own:
        ts = _framework()
        wrap = lambda x: ts.Tensor(x, device="hip")  # noqa: E731
        cache = ts.nn.PagedKVCache(case["batch"], case["kv_heads"], case["dim"], _capacity(case), device="hip",
                                   dtype=TORCH[case["dtype"]], page_size=PAGE)
        for i in range(0, n, chunk):
            cache.append(*(wrap(x[:, :, i:i + chunk]) for x in past))
        cache.truncate(got["lens"])
        state.update(cache=cache, ts=ts)
        state.update({name: wrap(got[name]) for name in ("q",) if name in got})
        state.update({name: [wrap(x) for x in got[name]] for name in ("new",) if name in got})
        return state
    pool = _Pool(case["batch"], case["kv_heads"], case["dim"], -(-_capacity(case) // PAGE))
    for i in range(0, n, chunk):
        rows = [x[:, :, i:i + chunk] for x in past]
        pool.write(rows, torch.arange(i, i + rows[0].shape[2], device=DEV).expand(case["batch"], -1))
    state.update(pool=pool, lens_dev=torch.tensor(got["lens"], device=DEV))
    state.update({name: got[name] for name in ("q", "new") if name in got})
    if case.get("rotary"):
        state["cos"], state["sin"] = _angles(case, _capacity(case))
    return state


def _own(state):
    case, cache, nn = state["case"], state["cache"], state["ts"].nn
    if case["kind"] == "attend":
        with state["ts"].no_grad():
            return nn.paged_attention(state["q"], cache)._data
    if case["kind"] == "append":
        cache.truncate(state["lens"])
        cache.append(*state["new"], rotary_base=10000.0 if case["rotary"] else None)
        return [x._data for x in cache.get(last=case["tokens"])]
    if case["kind"] == "fork":
        n = state["lens"][0]
        cache.truncate([n] * case["batch"])
        cache.reorder([0] * case["batch"])
        cache.append(*state["new"])
        return [x._data for x in cache.get(last=min(n + 1, PAGE))]
    return [x._data for x in cache.copy().get()]


def run(state):
    if own:
        return _own(state)
    return {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork,
            "copy": _plain_copy}[state["case"]["kind"]](state)


def work(case):
    es, d = SIZE[case["dtype"]], case["dim"]
    held = lambda positions: positions * case["kv_heads"] * d * 2 * BITS / 8  # noqa: E731
    lens, b = _lengths(case, 0), case["batch"]
    if case["kind"] == "attend":
        t, h = case["tokens"], case["heads"]
        pairs = sum(t * n - t * (t - 1) // 2 for n in lens)
        return {"bytes": int(held(sum(lens)) + 2 * b * h * t * d * es), "flops": 4 * pairs * h * d}
    values = lambda positions: positions * case["kv_heads"] * d * 2 * es  # noqa: E731
    if case["kind"] == "append":  # rows in, codes out, and their values read back
        n = b * case["tokens"]
        return {"bytes": int(2 * values(n) + held(n)), "flops": 8 * n * case["kv_heads"] * d}
    if case["kind"] == "fork":
        last, part = min(lens[0] + 1, PAGE), lens[0] % PAGE
        return {"bytes": int(values(b) + held((b - 1) * 2 * part) + held(b) + held(b * last) + values(b * last)),
                "flops": 2 * b * last * case["kv_heads"] * d}
    return {"bytes": int(2 * held(sum(lens)) + values(b * max(lens))), "flops": 2 * sum(lens) * case["kv_heads"] * d}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------


def _stored(x):
    """The values that the format keeps of rows x [..., D], in 64 bits."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    quotient = (g.abs().max(-1, keepdim=True).values / 6).float().double()  # fp32 by definition
    mantissa, exponent = torch.frexp(quotient)
    s = torch.ldexp(torch.round(mantissa * 64) / 64, exponent)
    s = torch.clamp(s, LEAST, MOST[x.dtype])
    borders = torch.tensor([b for b, _ in BORDERS], dtype=torch.float64, device=x.device)
    y = (g / s).abs()
    low, high = torch.bucketize(y, borders), torch.bucketize(y, borders, right=True)
    code = torch.where(low % 2 == 0, low, high)
    value = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[code] * s
    return torch.where(g < 0, -value, value).reshape(x.shape)


def _turned(k, first, case):
    """Keys [H, T, D] of one row rotated at positions first .., each operation rounded to the dtype."""
    t, d = k.shape[1], k.shape[2]
    freqs = 10000.0 ** (-np.arange(0, d, 2, dtype=np.float32) / np.float32(d))
    at = np.arange(first, first + t, dtype=np.float32)[:, None] * freqs
    c, s = (torch.from_numpy(f(at)).to(k.device).to(k.dtype).double() for f in (np.cos, np.sin))
    step = lambda z: z.to(k.dtype).double()  # noqa: E731
    x, y = k.double()[..., ::2], k.double()[..., 1::2]
    out = torch.empty_like(k)
    out[..., ::2] = (step(x * c) + step(-y * s)).to(k.dtype)
    out[..., 1::2] = (step(y * c) + step(x * s)).to(k.dtype)
    return out


def exact(case, seed):
    got = _inputs(case, seed)
    lens, d, dev = got["lens"], case["dim"], DEV
    if case["kind"] == "attend":
        t, hkv, out = case["tokens"], case["kv_heads"], []
        for b, n in enumerate(lens):
            k, v = (_stored(x[b, :, :n]) for x in got["past"])
            q = got["q"][b].double().view(hkv, -1, t, d)
            parts = []
            for h in range(hkv):
                x = q[h].reshape(-1, d) @ k[h].t() / math.sqrt(d)
                hidden = torch.arange(n, device=dev)[None] > torch.arange(n - t, n, device=dev)[:, None]
                x = x.view(-1, t, n).masked_fill(hidden, -math.inf)
                parts.append(torch.softmax(x, -1) @ v[h])
            out.append(torch.cat(parts))
        return torch.stack(out)
    if case["kind"] == "append":
        k, v = got["new"]
        if case["rotary"]:
            k = torch.stack([_turned(k[b], n, case) for b, n in enumerate(lens)])
        return [_stored(k), _stored(v)]
    if case["kind"] == "fork":
        n = lens[0]
        out = []
        for past, new in zip(got["past"], got["new"]):
            old = _stored(past[:1, :, :n]).expand(case["batch"], -1, -1, -1)
            out.append(torch.cat((old, _stored(new)), 2)[:, :, -PAGE:])
        return out
    out = []
    for x in got["past"]:
        y = torch.zeros(x.shape, dtype=torch.float64, device=dev)
        for b, n in enumerate(lens):
            y[b, :, :n] = _stored(x[b, :, :n])
        out.append(y)
    return out
