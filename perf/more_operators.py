"""Attention with a sliding window and sinks, attention of a tree of drafted tokens over a
cache, and the log probabilities of given tokens.

A case is a dict of plain values; ``kind`` says what one pass does:

* ``score``: ``functional.token_log_probs`` under ``no_grad``: log probabilities of given
  tokens, the rows' entropies and their ``top`` most likely tokens;
* ``learn``: the same with gradients of the log probabilities and entropies, back to the
  logits; a share of the rows is padding (``ignore_index``);
* ``window``: causal ``scaled_dot_product_attention`` whose queries see the last ``window``
  keys and the first ``sinks``, then ``backward`` with an upstream gradient;
* ``step``: ``cached_attention`` of the newest tokens over a key/value cache, through such
  a window;
* ``tree``: one round of drafted tokens: ``KVCache.append_tree`` (keys rotated at their
  depths' positions), ``cached_attention`` in which a token sees the cache and its own
  ancestors, and ``KVCache.keep`` of an accepted path, whose keys and values are read back.

A position's rotary angle is the product in fp32 of the position and its channel's
frequency, its cosine and sine rounded to the tensors' dtype, as are each product and sum
of the rotation; int8 caches hold ``round(x / s)`` with ``s = max(max|x| / 127, 1e-8)`` in
fp32 for each row.
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
IGNORED = -100
BASE = 10000.0


def _framework():
    path = os.path.join(os.getcwd(), "custom-ml-library_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tensorsmith_hip as ts

    return ts


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _score(name, dtype, rows, vocab, top):
    case = {"kind": "score", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top}
    return {"name": name, **case} if name else case


def _learn(name, dtype, rows, vocab, ignored):
    case = {"kind": "learn", "dtype": dtype, "rows": rows, "vocab": vocab, "top": 0, "ignored": ignored}
    return {"name": name, **case} if name else case


def _window(name, dtype, batch, heads, kv_heads, seq, dim, window, sinks):
    case = {"kind": "window", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq": seq,
            "dim": dim, "window": window, "sinks": sinks}
    return {"name": name, **case} if name else case


def _step(name, dtype, batch, heads, kv_heads, tokens, keys, dim, window, sinks):
    case = {"kind": "step", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens,
            "keys": keys, "dim": dim, "int8": False, "window": window, "sinks": sinks, "shared": True}
    return {"name": name, **case} if name else case


def _tree(name, dtype, batch, heads, kv_heads, tokens, keys, dim, int8, shared):
    case = {"kind": "tree", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens,
            "keys": keys, "dim": dim, "int8": int8, "shared": shared}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one sampled token with its five most likely alternatives: launches and host work count
        _score("score_f16_n1_v32000_top5", "f16", 1, 32000, 5),
        # a batch's step over a large vocabulary, twenty alternatives a token
        _score("score_bf16_n64_v128000_top20", "bf16", 64, 128000, 20),
        # the answers' tokens of a batch, with the entropies' gradient; an odd vocabulary
        _learn("learn_bf16_n8192_v50021", "bf16", 8192, 50021, 0.2),
        # the default dtype, a small vocabulary of odd size
        _learn("learn_f32_n777_v1009", "f32", 777, 1009, 0.1),
        # a long document with grouped-query heads
        _window("window_bf16_b2h16kv4_s8192_w1024", "bf16", 2, 16, 4, 8192, 128, 1024, 4),
        # odd lengths, a window that starts inside a tile, sinks past one tile
        _window("window_f16_b3h8_s2501_w300_d64", "f16", 3, 8, 8, 2501, 64, 300, 70),
        # the default dtype, a short sequence
        _window("window_f32_b2h4_s777_w100_d64", "f32", 2, 4, 4, 777, 64, 100, 3),
        # serving: a new token a sequence, half of the cache in its window
        _step("step_f16_b32h32kv8_k8192_w4096", "f16", 32, 32, 8, 1, 8192, 128, 4096, 4),
        # the smallest draft: five tokens of one stream
        _tree("tree_f16_b1h8_t5_k200_d64", "f16", 1, 8, 8, 5, 200, 64, False, True),
        # sixty-three drafted tokens a sequence, each sequence its own tree
        _tree("tree_bf16_b16h32kv8_t63_k8000", "bf16", 16, 32, 8, 63, 8000, 128, False, False),
        # over an int8 cache
        _tree("tree_int8_f16_b7h16kv4_t24_k4001", "f16", 7, 16, 4, 24, 4001, 128, True, False),
        # the default model's heads (4 of 32 channels) and dtype
        _tree("tree_f32_b8h4_t17_k900_d32", "f32", 8, 4, 4, 17, 900, 32, False, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    pick = rng.random()
    if pick < 0.2:
        rows, vocab = _log(rng, 1, 1000), _log(rng, 40, 200000)
        rows = max(1, min(rows, 64 * 128000 // vocab))
        return _score(None, dtype, rows, vocab, rng.choice([0, 1, 5, 20, min(vocab, 32)]))
    if pick < 0.4:
        rows, vocab = _log(rng, 1, 20000), _log(rng, 40, 200000)
        rows = max(1, min(rows, 8192 * 50021 // vocab // (2 if dtype == "f32" else 1)))
        return _learn(None, dtype, rows, vocab, rng.choice([0.0, 0.1, 0.5]))
    kv_heads, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 7, 8])
    if pick < 0.6:
        dim, seq, batch = rng.choice([32, 64, 128, 128]), _log(rng, 1, 8192), _log(rng, 1, 8)
        while batch * kv_heads * rep * seq * seq > (5e7 if dtype == "f32" else 2 * 16 * 8192 * 8192):
            if batch > 1:
                batch //= 2
            elif rep > 1:
                rep = 1
            else:
                seq //= 2
        window = _log(rng, 1, seq)
        return _window(None, dtype, batch, kv_heads * rep, kv_heads, seq, dim, window, rng.choice([0, 1, 4, 40, 130]))
    dim, keys, batch = rng.choice([32, 64, 128, 128]), _log(rng, 1, 16000), _log(rng, 1, 32)
    if pick < 0.75:
        tokens = rng.choice([1, 1, 1, 2, 5, 16])
        keys = max(keys, tokens)
        while batch * kv_heads * keys * dim > 32 * 8 * 8192 * 128 or batch * kv_heads * rep * tokens * keys > 1e8:
            batch, keys = max(1, batch // 2), max(tokens, keys // 2) if batch == 1 else keys
        return _step(None, dtype, batch, kv_heads * rep, kv_heads, tokens, keys, dim, _log(rng, 1, keys),
                     rng.choice([0, 1, 4, 40]))
    tokens = _log(rng, 1, 128)
    while batch * kv_heads * rep * tokens * (keys + tokens) > 16 * 32 * 63 * 8063:
        batch, tokens = max(1, batch // 2), max(1, tokens // 2) if batch == 1 else tokens
    int8 = dtype != "f32" and rng.random() < 0.3
    return _tree(None, dtype, batch, kv_heads * rep, kv_heads, tokens, keys, dim, int8, rng.random() < 0.4)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(case, seed):
    """Logits [N, V] with a few likely tokens a row and, at the end, vocabulary that no token uses; tokens, mostly
    likely ones; upstream gradients."""
    gen, n, v, dtype = _gen(seed), case["rows"], case["vocab"], TORCH[case["dtype"]]
    z = torch.randn((n, v), generator=gen, device=DEV, dtype=dtype).mul_(1.5)
    likely = torch.randint(0, v, (n, 3), generator=gen, device=DEV)
    z.scatter_add_(1, likely, (8 * torch.rand((n, 3), generator=gen, device=DEV)).to(dtype))
    if v > 100:
        z[:, v - v // 100:] = -math.inf
    some = torch.randint(0, v - v // 100, (n,), generator=gen, device=DEV)
    likely = torch.where(likely[:, 0] < v - v // 100, likely[:, 0], some)
    y = torch.where(torch.rand(n, generator=gen, device=DEV) < 0.7, likely, some)
    got = {"logits": z}
    if case["kind"] == "learn":
        y[torch.rand(n, generator=gen, device=DEV) < case["ignored"]] = IGNORED
        got["up"] = (torch.randn(n, generator=gen, device=DEV), 0.1 * torch.randn(n, generator=gen, device=DEV))
    got["tokens"] = y
    return got


def _operands(case, seed):
    """q, k, v and the upstream gradient, [B, H, S, D] as a layer has them: permuted projections."""
    gen, b, s, d, dtype = _gen(seed), case["batch"], case["seq"], case["dim"], TORCH[case["dtype"]]
    make = lambda h: torch.randn((b, s, h, d), generator=gen, device=DEV, dtype=dtype).permute(0, 2, 1, 3)  # noqa: E731
    h, hkv = case["heads"], case["kv_heads"]
    return {"q": make(h), "k": make(hkv), "v": make(hkv), "up": make(h)}


def _parents(case, seed):
    """Each drafted token's parent, -1 for the cache's last token, [B or 1, T]; and an accepted path [B, n], the
    same number for each row.  (The other tokens hang on any earlier one.)"""
    rng, t, b = np.random.default_rng(seed), case["tokens"], 1 if case["shared"] else case["batch"]
    n = max(1, t // 4)
    parents = np.floor(rng.random((b, t)) * (np.arange(t) + 1)).astype(np.int64) - 1
    path = np.sort(np.argsort(rng.random((b, t)), axis=1)[:, :n], axis=1)
    np.put_along_axis(parents, path, np.concatenate((np.full((b, 1), -1), path[:, :-1]), axis=1), axis=1)
    return parents, np.ascontiguousarray(np.broadcast_to(path, (case["batch"], n)))


def _ancestors(parents):
    """[B, T, T]: whether token s is t or one of its ancestors (the sum of the parent relation's powers)."""
    t = parents.shape[1]
    one = parents[..., None] == np.arange(t)
    return np.linalg.inv(np.eye(t) - one).round().astype(bool)


def _cached(case, seed):
    """The cache's keys (of unequal channels) and values before the pass, the new tokens' rows, and the tree."""
    gen, b, t, d, dtype = _gen(seed), case["batch"], case["tokens"], case["dim"], TORCH[case["dtype"]]
    make = lambda h, n: torch.randn((b, n, h, d), generator=gen, device=DEV, dtype=dtype).permute(0, 2, 1, 3)  # noqa: E731
    channels = torch.exp(0.5 * torch.randn(d, generator=gen, device=DEV)).to(dtype)
    got = {"past": (make(case["kv_heads"], case["keys"]) * channels, make(case["kv_heads"], case["keys"])),
           "q": make(case["heads"], t)}
    if case["kind"] == "tree":
        got["new"] = (make(case["kv_heads"], t) * channels, make(case["kv_heads"], t))
        got["parents"], got["path"] = _parents(case, seed)
    return got


def _angles(case, positions):
    """cos and sin [..., D / 2] of the rotary embedding at the positions, in the tensors' dtype."""
    d = case["dim"]
    freqs = BASE ** (-np.arange(0, d, 2, dtype=np.float32) / np.float32(d))
    at = positions.astype(np.float32)[..., None] * freqs
    return [torch.from_numpy(np.ascontiguousarray(f(at))).to(DEV, TORCH[case["dtype"]]) for f in (np.cos, np.sin)]


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------


def _plain_score(state):
    case, y = state["case"], state["tokens"]
    z = state["logits"].float()
    read = y != IGNORED
    m = z.amax(-1, keepdim=True)
    x = z - m
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    ln = torch.log(total)
    logp = (x.gather(1, torch.where(read, y, 0)[:, None]) - ln)[:, 0]
    entropy = ln[:, 0] - torch.where(e > 0, e * x, 0.0).sum(-1) / total[:, 0]
    out = {"log_probs": torch.where(read, logp, 0.0), "entropy": torch.where(read, entropy, 0.0)}
    if case["top"]:
        values, index = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_log_probs"] = (values - ln)[:, :case["top"]].contiguous()
        out["top_indices"] = index[:, :case["top"]].contiguous()
    if case["kind"] == "learn":
        g, gh = (torch.where(read, u, 0.0)[:, None] for u in state["up"])
        p, lnp = e / total, x - ln
        d = -p * g - gh * torch.where(p > 0, p * (lnp + entropy[:, None]), 0.0)
        d.scatter_add_(1, torch.where(read, y, 0)[:, None], g)
        out["gradient"] = d.to(state["logits"].dtype)
    return out


def _band(queries, keys, offset, window, sinks):
    """[Q, K]: whether query i, at position i + offset, sees key j."""
    i, j = torch.arange(queries, device=DEV)[:, None] + offset, torch.arange(keys, device=DEV)
    return (j <= i) & ((j < sinks) | (j > i - window))


def _plain_window(state):
    case = state["case"]
    b, h, s, d = state["q"].shape
    hkv, scale = case["kv_heads"], 1 / math.sqrt(d)
    rows = lambda x: x.float().reshape(b, hkv, -1, d)  # noqa: E731
    q, up = rows(state["q"]), rows(state["up"])
    k, v = state["k"].float().contiguous(), state["v"].float().contiguous()
    seen = _band(s, s, 0, case["window"], case["sinks"])
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(scale)
    x = x.view(b, h, s, s).masked_fill_(~seen, -math.inf)
    p = torch.exp_(x.sub_(x.amax(-1, keepdim=True)))
    p = p.div_(p.sum(-1, keepdim=True)).view(b, hkv, -1, s)
    out = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), up)
    delta = (up * out).sum(-1, keepdim=True)
    ds = torch.matmul(up, v.transpose(-1, -2).contiguous()).sub_(delta).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    t = state["q"].dtype
    return [out.view(b, h, s, d).to(t), dq.view(b, h, s, d).to(t), dk.to(t), dv.to(t)]


def _rotate(x, cos, sin):
    """Interleaved pairs by each row's angles; every product and sum rounds to x's dtype."""
    t = x.dtype
    r = lambda z: z.to(t).float()  # noqa: E731
    even, odd, c, s = x[..., 0::2].float(), x[..., 1::2].float(), cos.float(), sin.float()
    return torch.stack((r(r(even * c) - r(odd * s)), r(r(odd * c) + r(even * s))), -1).flatten(-2).to(t)


def _quantise(x):
    """Codes and scales of rows [..., D]."""
    x = x.float()
    s = (x.abs().amax(-1, keepdim=True).double() / 127).float().clamp(min=1e-8)
    return torch.round(x / s).to(torch.int8), s


def _held(state, side, at):
    """The fp32 values of positions `at` of the cache."""
    x = state["cache"][side][:, :, at].float()
    return x * state["scales"][side][:, :, at] if state["case"]["int8"] else x


def _store(state, rows, at):
    """Rows (keys, values) to positions `at` of the cache."""
    if state["case"]["int8"]:
        (kc, ks), (vc, vs) = _quantise(rows[0]), _quantise(rows[1])
        state["cache"][0][:, :, at], state["cache"][1][:, :, at] = kc, vc
        state["scales"][0][:, :, at], state["scales"][1][:, :, at] = ks, vs
    else:
        state["cache"][0][:, :, at], state["cache"][1][:, :, at] = rows


def _plain_attend(state, n, seen):
    """The new tokens' attention over the cache's first n positions; seen [B or 1, T, n]."""
    q = _rotate(state["q"], state["cos"][:, None], state["sin"][:, None])
    b, h, t, d = q.shape
    k, v = _held(state, 0, slice(0, n)), _held(state, 1, slice(0, n))
    hkv = k.shape[1]
    x = torch.matmul(q.float().reshape(b, hkv, -1, d), k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(d))
    x = x.view(b, h, t, n).masked_fill_(~seen[:, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hkv, -1, n), v.contiguous()).view(b, h, t, d)
    return (out / total).to(q.dtype)


def _plain_step(state):
    case = state["case"]
    n, t = case["keys"], case["tokens"]
    return _plain_attend(state, n, _band(t, n, n - t, case["window"], case["sinks"])[None])


def _plain_tree(state):
    case, path = state["case"], state["path"]
    first, t = case["keys"], case["tokens"]
    k, v = state["new"]
    _store(state, (_rotate(k, state["cos"][:, None], state["sin"][:, None]), v), slice(first, first + t))
    seen = state["ancestors"]
    past = torch.ones((seen.shape[0], t, first), dtype=torch.bool, device=DEV)
    out = _plain_attend(state, first + t, torch.cat((past, seen), -1))
    n, arrays = path.shape[1], state["cache"] + state["scales"]
    rows = [x[:, :, first:first + t].gather(2, path[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3]))
            for x in arrays]
    kept = slice(first, first + n)
    [x[:, :, kept].copy_(r) for x, r in zip(arrays, rows)]
    return [out, *(_held(state, side, kept).to(out.dtype) for side in (0, 1))]


# ---------------------------------------------------------------------------
# Entry points
# ---------------------------------------------------------------------------


def prepare(case, seed):
    if case["kind"] in ("score", "learn"):
        got = _logits(case, seed)
    elif case["kind"] == "window":
        got = _operands(case, seed)
    else:
        got = _cached(case, seed)
    state = {"case": case}
    if own:
        ts = _framework()
        wrap = lambda x: ts.Tensor(x, device="hip")  # noqa: E731
        state["ts"] = ts
        if case["kind"] == "learn":
            state["logits"] = ts.Tensor(got["logits"], device="hip", requires_grad=True)
            state["up"], state["tokens"] = [wrap(u) for u in got["up"]], wrap(got["tokens"])
        elif case["kind"] == "window":
            state["leaves"] = [ts.Tensor(got[name], device="hip", requires_grad=True) for name in ("q", "k", "v")]
            state["up"] = wrap(got["up"])
        elif case["kind"] == "score":
            state.update({name: wrap(x) for name, x in got.items()})
        else:
            room = case["keys"] + (case["tokens"] if case["kind"] == "tree" else 0)
            cache = ts.nn.KVCache(case["batch"], case["kv_heads"], case["dim"], room, device="hip",
                                  dtype=TORCH[case["dtype"]], quantized=case["int8"])
            with ts.no_grad():
                cache.append(*(wrap(x) for x in got["past"]))
            state.update(cache=cache, q=wrap(got["q"]))
            if case["kind"] == "tree":
                parents = got["parents"][0] if case["shared"] else got["parents"]
                state.update(new=[wrap(x) for x in got["new"]], path=wrap(torch.from_numpy(got["path"])),
                             tree=ts.nn.DraftTree(parents, device="hip"))
        return state
    state.update(got)
    if case["kind"] in ("step", "tree"):
        b, hkv, d, t = case["batch"], case["kv_heads"], case["dim"], case["tokens"]
        tree = case["kind"] == "tree"
        room = case["keys"] + (t if tree else 0)
        state["cache"] = [torch.zeros((b, hkv, room, d), dtype=torch.int8 if case["int8"] else TORCH[case["dtype"]],
                                      device=DEV) for _ in range(2)]
        state["scales"] = [torch.ones((b, hkv, room, 1), device=DEV) for _ in range(2)] if case["int8"] else []
        _store(state, got["past"], slice(0, case["keys"]))
        if tree:
            above = _ancestors(got["parents"])
            state["ancestors"], state["path"] = torch.from_numpy(above).to(DEV), torch.from_numpy(got["path"]).to(DEV)
            state["cos"], state["sin"] = _angles(case, case["keys"] + above.sum(-1) - 1)
        else:
            state["cos"], state["sin"] = _angles(case, np.arange(case["keys"] - t, case["keys"])[None])
    return state


def _own(state):
    case, ts = state["case"], state["ts"]
    if case["kind"] == "score":
        with ts.no_grad():
            got = ts.nn.functional.token_log_probs(state["logits"], state["tokens"], case["top"])
        out = {"log_probs": got.log_probs._data, "entropy": got.entropy._data}
        if case["top"]:
            out.update(top_log_probs=got.top_log_probs._data, top_indices=got.top_indices._data)
        return out
    if case["kind"] == "learn":
        z = state["logits"]
        z.zero_grad()
        got = ts.nn.functional.token_log_probs(z, state["tokens"])
        loss = (got.log_probs * state["up"][0] + got.entropy * state["up"][1]).sum()
        loss.backward()
        return {"log_probs": got.log_probs._data, "entropy": got.entropy._data, "gradient": z._grad}
    if case["kind"] == "window":
        q, k, v = state["leaves"]
        q.zero_grad(), k.zero_grad(), v.zero_grad()
        out = ts.nn.scaled_dot_product_attention(q, k, v, is_causal=True, window=case["window"], sinks=case["sinks"],
                                                 enable_gqa=True)
        out.backward(state["up"])
        return [out._data, q._grad, k._grad, v._grad]
    cache = state["cache"]
    with ts.no_grad():
        if case["kind"] == "step":
            return ts.nn.cached_attention(state["q"], cache, window=case["window"], sinks=case["sinks"],
                                          rotary_base=BASE)._data
        cache.truncate(case["keys"])
        cache.append_tree(*state["new"], state["tree"], rotary_base=BASE)
        out = ts.nn.cached_attention(state["q"], cache, state["tree"], rotary_base=BASE)
        cache.keep(case["keys"], state["path"])
        return [out._data, *(x._data for x in cache.get(last=state["path"].shape[1]))]


def run(state):
    if own:
        return _own(state)
    return {"score": _plain_score, "learn": _plain_score, "window": _plain_window, "step": _plain_step,
            "tree": _plain_tree}[state["case"]["kind"]](state)


def work(case):
    es = SIZE[case["dtype"]]
    if case["kind"] in ("score", "learn"):
        n, v = case["rows"], case["vocab"]
        small = n * (8 + 8 + 12 * case["top"])
        if case["kind"] == "score":
            return {"bytes": n * v * es + small, "flops": 6 * n * v}
        return {"bytes": 2 * n * v * es + small + 8 * n, "flops": 14 * n * v}
    b, h, hkv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "window":
        s, w, sinks = case["seq"], case["window"], case["sinks"]
        i = np.arange(s)
        pairs = int((np.minimum(i + 1, w) + np.minimum(np.maximum(i + 1 - w, 0), sinks)).sum())
        # q, out, its gradient and dq; k, v, dk and dv
        return {"bytes": b * s * d * es * 4 * (h + hkv), "flops": 14 * b * h * pairs * d}
    held = hkv * d * 2 * (1 if case["int8"] else es) + (hkv * 8 if case["int8"] else 0)  # a position's
    t, n = case["tokens"], case["keys"]
    io = 2 * b * h * t * d * es
    if case["kind"] == "step":
        w, sinks = case["window"], case["sinks"]
        seen = min(n, w + t - 1) + min(sinks, max(0, n - (w + t - 1)))
        return {"bytes": b * seen * held + io, "flops": 4 * b * h * t * min(n, w + sinks) * d}
    new, kept = b * t * hkv * d * 2 * es, max(1, t // 4)
    # the cache and the new rows read, the new rows held; the path's rows moved and read back
    return {"bytes": b * (n + t) * held + io + new + b * t * held + 2 * b * kept * held + b * kept * hkv * d * 2 * es,
            "flops": 4 * b * h * t * n * d}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------


def _turned(x, positions, case):
    """Rows [B, H, T, D] rotated at positions [B, T], each operation rounded to the dtype."""
    d = case["dim"]
    freqs = BASE ** (-np.arange(0, d, 2, dtype=np.float32) / np.float32(d))
    at = positions.astype(np.float32)[..., None] * freqs
    c, s = (torch.from_numpy(f(at)).to(x.device).to(x.dtype).double()[:, None] for f in (np.cos, np.sin))
    step = lambda z: z.to(x.dtype).double()  # noqa: E731
    u, w = x.double()[..., ::2], x.double()[..., 1::2]
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out[..., ::2] = (step(u * c) + step(-w * s)).to(x.dtype)
    out[..., 1::2] = (step(w * c) + step(u * s)).to(x.dtype)
    return out


def _kept(x, int8):
    """The values that a cache holds of rows [..., D], in 64 bits."""
    if not int8:
        return x.double()
    s = (x.double().abs().max(-1, keepdim=True).values / 127).float().clamp(min=1e-8).double()
    return torch.round(x.double() / s) * s


def exact(case, seed):
    if case["kind"] in ("score", "learn"):
        got = _logits(case, seed)
        y, top, out = got["tokens"], case["top"], []
        for i in range(0, case["rows"], 1024):  # (rows a part: 64 bits of all logits are many)
            z, t = got["logits"][i:i + 1024].double(), y[i:i + 1024]
            live, at = t != IGNORED, t.clamp(min=0)[:, None]
            lp = torch.log_softmax(z, -1)
            p = torch.exp(lp)
            surprise = torch.where(p > 0, lp, 0.0)
            entropy = -(p * surprise).sum(-1)
            part = {"log_probs": lp.gather(1, at)[:, 0] * live, "entropy": entropy * live}
            if top:
                index = torch.argsort(lp, dim=-1, descending=True, stable=True)[:, :top]
                part["top_log_probs"], part["top_indices"] = lp.gather(1, index), index
            if case["kind"] == "learn":
                g, gh = (u[i:i + 1024].double() * live for u in got["up"])
                hot = torch.zeros_like(p).scatter_(1, at, 1.0)
                part["gradient"] = g[:, None] * (hot - p) - gh[:, None] * p * (surprise + entropy[:, None])
            out.append(part)
        return {name: torch.cat([part[name] for part in out]) for name in out[0]}
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    scale = 1 / math.sqrt(d)
    if case["kind"] == "window":
        got = _operands(case, seed)
        s, rep = case["seq"], h // hkv
        i, j = torch.arange(s, device=DEV)[:, None], torch.arange(s, device=DEV)[None]
        hidden = (j > i) | ((j >= case["sinks"]) & (i - j >= case["window"]))
        out = [torch.zeros(x.shape, dtype=torch.float64, device=DEV)
               for x in (got["q"], got["q"], got["k"], got["v"])]
        for b in range(case["batch"]):
            for n in range(h):
                q, up = got["q"][b, n].double(), got["up"][b, n].double()
                k, v = got["k"][b, n // rep].double(), got["v"][b, n // rep].double()
                p = torch.softmax((q @ k.t() * scale).masked_fill_(hidden, -math.inf), -1)
                o = p @ v
                ds = (up @ v.t() - (up * o).sum(-1, keepdim=True)) * p * scale
                out[0][b, n], out[1][b, n] = o, ds @ k
                out[2][b, n // rep] += ds.t() @ q
                out[3][b, n // rep] += p.t() @ up
        return out
    got = _cached(case, seed)
    b, t, n, int8 = case["batch"], case["tokens"], case["keys"], case["int8"]
    k, v = (_kept(x, int8) for x in got["past"])
    if case["kind"] == "step":
        at = np.broadcast_to(np.arange(n - t, n), (b, t))
        i, j = torch.arange(n - t, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        hidden = ((j > i) | ((j >= case["sinks"]) & (i - j >= case["window"]))).expand(b, t, n)
    else:
        above = np.broadcast_to(_ancestors(got["parents"]), (b, t, t))
        at = n + above.sum(-1) - 1
        new = [_kept(x, int8) for x in (_turned(got["new"][0], at, case), got["new"][1])]
        k, v = torch.cat((k, new[0]), 2), torch.cat((v, new[1]), 2)
        hidden = torch.zeros((b, t, n + t), dtype=torch.bool, device=DEV)
        hidden[..., n:] = ~torch.from_numpy(above.copy()).to(DEV)
    q, out = _turned(got["q"], at, case).double(), []
    for r in range(b):
        x = (q[r].reshape(hkv, -1, d) @ k[r].transpose(-1, -2) * scale).view(h, t, -1)
        p = torch.softmax(x.masked_fill_(hidden[r], -math.inf), -1)
        out.append((p.view(hkv, -1, p.shape[-1]) @ v[r]).view(h, t, d))
    out = torch.stack(out)
    if case["kind"] == "step":
        return out
    path = torch.from_numpy(got["path"]).to(DEV)[:, None, :, None].expand(-1, hkv, -1, d)
    return [out, *(x.gather(2, path) for x in new)]
