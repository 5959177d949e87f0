"""Attention of new tokens over a key/value cache through a window or as a drafted tree,
the tree's plan, its append and the rows that are kept, against float64 and array
operations.

Bounds: over f16 and bf16 caches P rounds to the type (2^-11, 2^-8 a term at most, over int8
codes 2^-8 and for f16 queries 2^-16) and the result once (2^-11, 2^-8): at most 2^-7 of the
terms' sizes, and relative 2-norms of a row, whose roundings are independent, below 1e-2; in
f32 below 2e-5.  A key too many or too few moves a row by the order of
its size divided by the number of keys that it sees, which the short contexts make large.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("no GPU", allow_module_level=True)

import tensorsmith_hip as ts  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402

BOUND = {torch.float16: 1e-2, torch.bfloat16: 1e-2, torch.float32: 2e-5}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
BASE = 10000.0


def _wrap(x, grad=False):
    return ts.Tensor(x, device="hip", requires_grad=grad)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(b, h, n, d, dtype, seed):
    """[B, H, n, D] as a layer has them: a permuted view."""
    return torch.randn((b, n, h, d), generator=_gen(seed), device="cuda").to(dtype).permute(0, 2, 1, 3)


def _turn(x, positions):
    """RoPE of [B, H, T, D] at positions [B or 1, T], every product and sum rounded to the type."""
    d = x.shape[-1]
    freqs = BASE ** (-np.arange(0, d, 2, dtype=np.float32) / np.float32(d))
    at = np.asarray(positions, np.float32)[..., None] * freqs
    c, s = (torch.from_numpy(f(at)).cuda().to(x.dtype).double()[:, None] for f in (np.cos, np.sin))
    step = lambda z: z.to(x.dtype).double()  # noqa: E731
    u, w = x.double()[..., ::2], x.double()[..., 1::2]
    out = torch.empty_like(x)
    out[..., ::2] = (step(u * c) - step(w * s)).to(x.dtype)
    out[..., 1::2] = (step(w * c) + step(u * s)).to(x.dtype)
    return out


def _parents(rng, trees, tokens):
    return np.floor(rng.random((trees, tokens)) * (np.arange(tokens) + 1)).astype(np.int64) - 1


def _ancestors(parents):
    trees, tokens = parents.shape
    seen = np.zeros((trees, tokens, tokens), bool)
    for b in range(trees):
        for t in range(tokens):
            s = t
            while s >= 0:
                seen[b, t, s] = True
                s = parents[b, s]
    return seen


def _cache(b, hkv, n, d, dtype, int8=False, room=0, seed=0):
    cache = nn.KVCache(b, hkv, d, n + room, device="hip", dtype=dtype, quantized=int8)
    if n:
        with ts.no_grad():
            cache.append(_wrap(_rows(b, hkv, n, d, dtype, seed + 1)), _wrap(_rows(b, hkv, n, d, dtype, seed + 2)))
    return cache


def _values(cache):
    """The cached keys and values in float64, as they are held."""
    keys, values, ks, vs = cache.storage
    out = []
    for x, s in ((keys, ks), (values, vs)):
        x = x[:, :, :cache.length].double()
        out.append(x if s is None else x * s[:, :, :cache.length].double())
    return out


def _reference(q, cache, seen, scale=None):
    k, v = _values(cache)
    rep = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    x = torch.matmul(q.double(), k.transpose(-1, -2)) * (1 / math.sqrt(q.shape[-1]) if scale is None else scale)
    return torch.matmul(torch.softmax(x.masked_fill(~seen, -math.inf), -1), v)


def _close(got, want, dtype):
    err, size = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    bad = err > BOUND[dtype] * torch.maximum(size, 0.1 * size.square().mean().sqrt())
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (err / size).max().item())


def _attend(q, cache, *args, **kw):
    with ts.no_grad():
        return nn.cached_attention(_wrap(q), cache, *args, **kw)._data


def _band(tokens, n, window, sinks):
    i, j = torch.arange(n - tokens, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    return (j <= i) & ((j > i - window) | (j < sinks))


# (batch, KV heads, query heads a KV head, tokens, positions)
SIZES = [(1, 1, 1, 1, 1), (2, 2, 1, 1, 40), (1, 2, 4, 1, 700), (3, 1, 8, 2, 333), (1, 2, 7, 5, 129), (2, 1, 4, 17, 500),
         (1, 1, 3, 33, 65), (1, 2, 1, 100, 1000), (1, 1, 5, 64, 64), (2, 8, 4, 1, 3001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("size", SIZES)
def test_windows_match_float64(size, d, dtype):
    b, hkv, rep, tokens, n = size
    cache = _cache(b, hkv, n, d, dtype)
    q = _rows(b, hkv * rep, tokens, d, dtype, 7)
    for window, sinks in ((1, 0), (3, 1), (32, 0), (33, 40), (100, 4), (max(1, n // 2), 32), (n + 9, 3)):
        print("cached window", size, d, dtype, window, sinks, flush=True)
        got = _attend(q, cache, window=window, sinks=sinks)
        _close(got, _reference(q, cache, _band(tokens, n, window, sinks)), dtype)
    got = _attend(q, cache, scale=0.3)
    _close(got, _reference(q, cache, _band(tokens, n, n, 0), 0.3), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (2, 2, 4, 1, 333), (1, 2, 3, 5, 129), (3, 1, 4, 17, 1000),
                                  (1, 1, 2, 130, 400)])
def test_int8_caches_match_float64(size, d, dtype):
    b, hkv, rep, tokens, n = size
    cache = _cache(b, hkv, n, d, dtype, int8=True)
    q = _rows(b, hkv * rep, tokens, d, dtype, 8)
    for window, sinks in ((5, 0), (64, 33), (n, 0)):
        print("cached int8", size, d, dtype, window, sinks, flush=True)
        _close(_attend(q, cache, window=window, sinks=sinks), _reference(q, cache, _band(tokens, n, window, sinks)),
               dtype)


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 64, 100, 255, 256])
def test_trees_from_the_host_and_the_device(tokens):
    rng = np.random.default_rng(tokens)
    chain, star = np.arange(tokens)[None] - 1, np.full((1, tokens), -1)
    for parents in (_parents(rng, 3, tokens), chain, star):
        seen = _ancestors(parents)
        trees = [nn.DraftTree(parents), nn.DraftTree(_wrap(torch.from_numpy(parents).cuda())),
                 nn.DraftTree(_wrap(torch.from_numpy(parents.astype(np.int32)).cuda()))]
        for tree in trees:
            assert np.array_equal(tree._visible().cpu().numpy(), seen)
            assert np.array_equal(tree.depths.numpy(), seen.sum(-1) - 1)
    flat = nn.DraftTree(chain[0].tolist())
    assert flat.depths.numpy().tolist() == list(range(tokens)) and flat.trees == 1


def test_parents_that_are_no_earlier_token_count_as_none():
    raw = torch.tensor([5, -7, 0, 3, 2 ** 31 - 1, 1], device="cuda")
    tree = nn.DraftTree(_wrap(raw))
    want = _ancestors(np.array([[-1, -1, 0, -1, -1, 1]]))
    assert np.array_equal(tree._visible().cpu().numpy(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 0, 64), (2, 2, 4, 5, 200, 64), (3, 1, 4, 33, 77, 32),
                                  (2, 2, 2, 64, 1000, 128), (1, 2, 4, 100, 31, 128), (2, 1, 1, 256, 500, 64),
                                  (1, 1, 2, 20, 300, 256)])
def test_trees_match_float64(size, dtype):
    b, hkv, rep, tokens, n, d = size
    rng = np.random.default_rng(tokens)
    for int8 in (False, True):
        if int8 and dtype == torch.float32:
            continue
        for shared in (True, False):
            print("tree", size, dtype, int8, shared, flush=True)
            cache = _cache(b, hkv, n, d, dtype, int8=int8, room=tokens + 3)
            parents = _parents(rng, 1 if shared else b, tokens)
            tree = nn.DraftTree(parents[0] if shared else parents)
            k, v, q = (_rows(b, h, tokens, d, dtype, s) for h, s in ((hkv, 4), (hkv, 5), (hkv * rep, 6)))
            with ts.no_grad():
                cache.append_tree(_wrap(k), _wrap(v), tree, rotary_base=BASE)
            assert cache.length == n + tokens
            seen = torch.from_numpy(_ancestors(parents)).cuda()
            at = n + seen.sum(-1).cpu().numpy() - 1
            plain = _cache(b, hkv, n, d, dtype, int8=int8, room=tokens + 3)
            with ts.no_grad():
                plain.append(_wrap(_turn(k, at)), _wrap(v))
            for x, y in zip(cache.storage, plain.storage):
                assert x is None or torch.equal(x, y)
            past = torch.ones((seen.shape[0], tokens, n), dtype=torch.bool, device="cuda")
            turned = _turn(q, at)
            want = _reference(turned, cache, torch.cat((past, seen), -1)[:, None])
            _close(_attend(q, cache, tree, rotary_base=BASE), want, dtype)
            _close(_attend(turned, cache, tree), want, dtype)
            window, sinks = tokens + n // 3, 4
            j = torch.arange(n, device="cuda")
            past = (j > torch.from_numpy(at).cuda()[..., None] - window) | (j < sinks)
            want = _reference(turned, cache, torch.cat((past, seen), -1)[:, None])
            _close(_attend(q, cache, tree, rotary_base=BASE, window=window, sinks=sinks), want, dtype)


def test_what_the_kernel_does_not_take_goes_by_a_mask():
    rng = np.random.default_rng(1)
    for dtype, d, dv in ((torch.float64, 64, 64), (torch.float32, 256, 256), (torch.float16, 48, 48),
                         (torch.float16, 64, 128)):
        n, tokens = 90, 7
        cache = nn.KVCache(2, 2, d, n + tokens, device="hip", dtype=dtype, value_dim=dv)
        with ts.no_grad():
            cache.append(_wrap(_rows(2, 2, n, d, dtype, 1)), _wrap(_rows(2, 2, n, dv, dtype, 2)))
            tree = nn.DraftTree(_parents(rng, 2, tokens))
            k, v, q = _rows(2, 2, tokens, d, dtype, 3), _rows(2, 2, tokens, dv, dtype, 4), _rows(2, 4, tokens, d, dtype, 5)
            cache.append_tree(_wrap(k), _wrap(v), tree, rotary_base=BASE)
        seen = tree._visible()
        at = n + seen.sum(-1).cpu().numpy() - 1
        if dtype != torch.float64:  # (its tables are fp32's angles in 64 bits)
            assert torch.equal(cache.storage[0][:, :, n:], _turn(k, at))
        past = torch.ones((2, tokens, n), dtype=torch.bool, device="cuda")
        want = _reference(_turn(q, at), cache, torch.cat((past, seen), -1)[:, None])
        _close(_attend(q, cache, tree, rotary_base=BASE), want, torch.float32 if dtype == torch.float64 else dtype)
        got = _attend(q, cache, window=30, sinks=2)
        _close(got, _reference(q, cache, _band(tokens, n + tokens, 30, 2)), torch.float32 if dtype == torch.float64 else dtype)
    cache = _cache(1, 1, 700, 64, torch.float16)
    q = _rows(1, 2, 300, 64, torch.float16, 9)
    _close(_attend(q, cache, window=90, sinks=3), _reference(q, cache, _band(300, 700, 90, 3)), torch.float16)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16), (32, torch.float32), (20, torch.float16),
                                     (7, torch.float32), (3, torch.float16)])
def test_kept_rows(d, dtype, int8):
    rng = np.random.default_rng(d)
    for n, drafted, kept in ((0, 1, 1), (10, 9, 4), (33, 256, 256), (5, 100, 70), (5, 6, 0)):
        cache = _cache(3, 2, n + drafted, d, dtype, int8=int8, room=2)
        before = [None if x is None else x.clone() for x in cache.storage]
        index = np.stack([rng.permutation(drafted)[:kept] for _ in range(3)]) if kept else np.zeros((3, 0), np.int64)
        if kept > 2:
            index[1, 1] = index[1, 0]  # twice the same
        print("keep", d, dtype, int8, n, drafted, kept, flush=True)
        cache.keep(n, index if drafted % 2 else _wrap(torch.from_numpy(index.astype(np.int32)).cuda()))
        assert cache.length == n + kept
        at = torch.from_numpy(index).cuda()[:, None, :, None]
        for x, y in zip(cache.storage, before):
            if x is None:
                continue
            want = y.clone()
            if kept:
                want[:, :, n:n + kept] = y[:, :, n:].gather(2, at.expand(-1, 2, -1, y.shape[3]))
            assert torch.equal(x, want)


def test_kept_indices_out_of_range_leave_the_row():
    cache = _cache(1, 1, 12, 64, torch.float16)
    before = cache.storage[0].clone()
    cache.keep(4, _wrap(torch.tensor([[7, -1, 8, 2 ** 40, 3]], device="cuda")))
    want = before.clone()
    want[:, :, 4], want[:, :, 8] = before[:, :, 11], before[:, :, 7]
    assert torch.equal(cache.storage[0], want) and cache.length == 9


def test_rows_behind_the_cache_are_left_and_not_read():
    cache = _cache(2, 2, 300, 64, torch.float16, room=40)
    for x in cache.storage[:2]:
        x[:, :, 300:] = math.nan
    q = _rows(2, 4, 3, 64, torch.float16, 3)
    tree = nn.DraftTree([-1, 0, 0])
    assert torch.isfinite(_attend(q, cache, tree)).all() and torch.isfinite(_attend(q, cache, window=50, sinks=2)).all()
    with ts.no_grad():
        cache.append_tree(_wrap(_rows(2, 2, 3, 64, torch.float16, 4)), _wrap(_rows(2, 2, 3, 64, torch.float16, 5)), tree)
    assert torch.isnan(cache.storage[0][:, :, 303:]).all() and torch.isfinite(cache.storage[0][:, :, :303]).all()


def _model(window=None, sinks=0, dtype="float32"):
    ts.seed(11)
    model = nn.TransformerLM(nn.TransformerConfig(97, dim=128, num_heads=4, num_kv_heads=2, num_layers=2,
                                                  hidden_dim=256, max_seq_len=400, attention_window=window,
                                                  attention_sinks=sinks), device="hip").eval()
    return model if dtype == "float32" else model.to(dtype=dtype)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 3)])
def test_a_round_of_drafted_tokens_is_the_path_token_by_token(window, sinks, quantized):
    """A model's logits of a tree's nodes, and of what follows a kept path, are those of the path fed alone.
    Each layer rounds P and its results as the plain step does, in f32 (int8 caches: the same codes)."""
    model = _model(window, sinks)
    tokens = torch.randint(0, 97, (2, 150), device="cuda")
    drafted = torch.randint(0, 97, (2, 9), device="cuda")
    parents = np.array([-1, -1, 0, 1, 1, 2, 4, 6, 3])
    path = [1, 4, 6, 7]
    with ts.no_grad():
        caches = model.new_cache(2, quantized=quantized)
        model(_wrap(tokens), caches=caches, logits_to_keep=1)
        logits = model(_wrap(drafted), caches=caches, tree=nn.DraftTree(parents))._data
        score = nn.functional.token_log_probs(_wrap(logits[:, path[:-1]]), _wrap(drafted[:, path[1:]]), 3)
        for cache in caches:
            cache.keep(150, np.array([path, path]))
        after = model(_wrap(drafted[:, :1]), caches=caches)._data
        plain = model.new_cache(2, quantized=quantized)
        model(_wrap(tokens), caches=plain, logits_to_keep=1)
        steps = [model(_wrap(drafted[:, t:t + 1]), caches=plain)._data[:, 0] for t in path]
        last = model(_wrap(drafted[:, :1]), caches=plain)._data
    bound = 2e-2 if quantized else 1e-4
    for i, t in enumerate(path):
        assert (logits[:, t] - steps[i]).norm() <= bound * steps[i].norm(), t
    assert (after - last).norm() <= bound * last.norm()
    want = torch.log_softmax(torch.stack(steps[:-1], 1).double(), -1).gather(-1, drafted[:, path[1:]][..., None])[..., 0]
    assert (score.log_probs._data - want).abs().max() <= (0.2 if quantized else 1e-3)
    assert score.top_indices.shape == (2, 3, 3)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("quantized", [False, True])
def test_a_windowed_model_steps_as_it_trains(dtype, quantized):
    model = _model(40, 2, dtype)
    tokens = torch.randint(0, 97, (2, 130), device="cuda")
    with ts.no_grad():
        want = model(_wrap(tokens))._data
        caches = model.new_cache(2, quantized=quantized)
        got = [model(_wrap(tokens[:, :100]), caches=caches)._data]
        got += [model(_wrap(tokens[:, i:i + 1]), caches=caches)._data for i in range(100, 130)]
    bound = 2e-2 if quantized or dtype == "float16" else 1e-4
    assert (torch.cat(got, 1).double() - want.double()).norm() <= bound * want.double().norm()
    out = model.generate(_wrap(tokens[:, :50]), 20, temperature=0.0, quantized_cache=quantized)
    assert out.shape == (2, 70)


def test_a_captured_round_replays_and_another_stream_agrees():
    b, hkv, d, n, tokens = 2, 2, 128, 600, 12
    caches = [_cache(b, hkv, n, d, torch.bfloat16, room=tokens) for _ in range(2)]
    parents = _wrap(torch.from_numpy(_parents(np.random.default_rng(2), b, tokens)).cuda())
    path = _wrap(torch.tensor([[3, 1], [0, 11]], device="cuda"))
    k, v, q = (_rows(b, h, tokens, d, torch.bfloat16, s).clone() for h, s in ((hkv, 4), (hkv, 5), (8, 6)))

    def step(cache):
        with ts.no_grad():
            cache.truncate(n)
            tree = nn.DraftTree(parents)
            cache.append_tree(_wrap(k), _wrap(v), tree, rotary_base=BASE)
            out = nn.cached_attention(_wrap(q), cache, tree, rotary_base=BASE)._data
            cache.keep(n, path)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, step(caches[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for seed in range(3):
        for x, s in ((k, 14), (v, 15), (q, 16)):
            x.copy_(_rows(*x.shape[:2], tokens, d, torch.bfloat16, s + 10 * seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step(caches[1]))
        for x, y in zip(caches[0].storage[:2], caches[1].storage[:2]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 9, 20, 40])
def test_long_int8_caches_are_cut_in_parts(tokens, d, dtype):
    """Scales from 2^-8 to 2^8 of neighbouring rows, so that a code under another row's scale shows."""
    b, hkv, rep, n = 2, 3, 4, 4321
    cache = _cache(b, hkv, n, d, dtype, int8=True)
    for scales in cache.storage[2:]:
        scales *= 2.0 ** torch.randint(-8, 9, scales.shape, device="cuda")
    q = _rows(b, hkv * rep, tokens, d, dtype, 7) * 2.0 ** -8
    for window, sinks in ((4000, 0), (777, 65)):
        got = _attend(q, cache, window=window, sinks=sinks)
        _close(got, _reference(q, cache, _band(tokens, n, window, sinks)), dtype)
    parents = _parents(np.random.default_rng(tokens), b, tokens)
    seen = torch.ones(b, 1, tokens, n, dtype=torch.bool, device="cuda")
    seen[:, 0, :, n - tokens:] = torch.from_numpy(_ancestors(parents)).cuda()
    _close(_attend(q, cache, nn.DraftTree(parents)), _reference(q, cache, seen), dtype)


def test_scales_that_lie_apart_or_are_shared_by_rows():
    """Scales of a wider stride are read where they lie; one for all rows has no kernel and is dequantised."""
    b, hkv, n, d = 1, 2, 300, 64
    cache = _cache(b, hkv, n, d, torch.float16, int8=True)
    q = _rows(b, 4, 3, d, torch.float16, 7)
    want = _attend(q, cache, window=100)
    for name in ("_key_scales", "_value_scales"):
        apart = torch.full((b, hkv, n, 3), 1e30, device="cuda")
        apart[..., :1] = getattr(cache, name)
        setattr(cache, name, apart[..., :1])
    cache._described = ()
    assert torch.equal(_attend(q, cache, window=100), want)
    cache._key_scales = torch.full((b, hkv, 1, 1), 0.01, device="cuda").expand(b, hkv, n, 1)
    cache._described = ()
    _close(_attend(q, cache, window=100), _reference(q, cache, _band(3, n, 100, 0)), torch.float16)


def test_windows_over_a_paged_cache():
    """A window over all positions leaves the paged kernels on; a smaller one reads the values back."""
    x = _wrap(torch.randn(2, 50, 128, generator=_gen(3), device="cuda").half())
    layers = []
    for window in (None, 50, 20):
        ts.seed(5)
        layers.append(nn.MultiHeadAttention(128, 4, num_kv_heads=2, rotary=False, window=window, sinks=0 if window is None else 2,
                                            device="hip").eval().to(dtype="float16"))
    with ts.no_grad():
        got, caches = [], []
        for layer in layers:
            caches.append(nn.PagedKVCache(2, 2, 32, 64, device="hip", dtype="float16"))
            got.append([layer(x[:, :45], cache=caches[-1])._data, layer(x[:, 45:], cache=caches[-1])._data])
        for one, other in zip(got[0], got[1]):
            assert torch.equal(one, other)
        k, v = (y._data.double().repeat_interleave(2, 1) for y in caches[2].get())
        q = layers[2].q_proj(x)._data.double().reshape(2, 50, 4, 32).permute(0, 2, 1, 3)[:, :, 45:]
        s = (torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(32)).masked_fill(~_band(5, 50, 20, 2), -math.inf)
        want = torch.matmul(torch.softmax(s, -1), v).permute(0, 2, 1, 3).reshape(2, 5, 128)
        want = torch.matmul(want, layers[2].out_proj.weight._data.double().t().contiguous())
    assert (got[2][1].double() - want).norm() <= 1e-2 * want.norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("d,dv,n", [(128, 128, 300), (64, 32, 7), (8, 24, 1), (5, 3, 40), (16, 12, 33), (256, 256, 1000)])
def test_codes_are_read_as_products_rounded_once(d, dv, n, dtype):
    """The same bits as array operations: the product in float32, then the type."""
    b, h, room = 2, 3, n + 5
    cache = nn.KVCache(b, h, d, room, device="hip", dtype=dtype, quantized=True, value_dim=dv)
    for x in cache.storage[:2]:
        x.copy_(torch.randint(-127, 128, x.shape, device="cuda", generator=_gen(n)))
    for x in cache.storage[2:]:
        x.copy_(2.0 ** (20 * torch.rand(x.shape, device="cuda", generator=_gen(d)) - 14))
    cache.length = n
    for last in (None, 1, n // 2, 0):
        first = 0 if last is None else n - last
        for got, x, s in zip(cache.get(last), cache.storage[:2], cache.storage[2:]):
            want = (x[:, :, first:n].float() * s[:, :, first:n]).to(dtype)
            assert got.shape == want.shape and torch.equal(got._data, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("tokens,rep,n", [(33, 1, 33), (17, 4, 300), (128, 1, 517), (70, 3, 1000)])
def test_many_heads_share_their_tiles(tokens, rep, n, d, dtype):
    """128 heads or more: four waves of 32 rows to a tile, whole and cut rows, from one tile to several parts."""
    b, hkv = 16, 8
    cache = _cache(b, hkv, n, d, dtype)
    q = _rows(b, hkv * rep, tokens, d, dtype, 7)
    parents = _parents(np.random.default_rng(tokens), b, tokens)
    seen = torch.ones(b, 1, tokens, n, dtype=torch.bool, device="cuda")
    seen[:, 0, :, n - tokens:] = torch.from_numpy(_ancestors(parents)).cuda()
    print("shared tiles", tokens, rep, n, d, dtype, flush=True)
    _close(_attend(q, cache, nn.DraftTree(parents)), _reference(q, cache, seen), dtype)
    for window, sinks in ((1, 0), (31, 33), (n // 2, 3)):
        _close(_attend(q, cache, window=max(1, window), sinks=sinks),
               _reference(q, cache, _band(tokens, n, max(1, window), sinks)), dtype)


@pytest.mark.parametrize("tokens,rep,n,d,dtype,int8", [(1, 4, 8300, 128, torch.float16, False),
                                                       (12, 4, 8299, 128, torch.bfloat16, False),
                                                       (1, 8, 16501, 128, torch.bfloat16, True),
                                                       (3, 1, 8301, 64, torch.float32, False)])
def test_caches_larger_than_the_memory_side_cache(tokens, rep, n, d, dtype, int8):
    """Keys and values of more than 256 MB, which are read past it; three of the sequences are compared."""
    b, hkv = 16, 8
    cache = _cache(b, hkv, n, d, dtype, int8)
    q = _rows(b, hkv * rep, tokens, d, dtype, 7)
    for window, sinks in ((n - 77, 5), (n + 1, 0)):
        print("large caches", tokens, rep, n, d, dtype, int8, window, flush=True)
        got = _attend(q, cache, window=window, sinks=sinks)
        for i in (0, 7, 15):
            one = nn.KVCache(1, hkv, d, n, device="hip", dtype=dtype, quantized=int8)
            for x, y in zip(one.storage, cache.storage):
                if x is not None:
                    x.copy_(y[i:i + 1])
            one.length = n
            _close(got[i:i + 1], _reference(q[i:i + 1], one, _band(tokens, n, window, sinks)), dtype)


@pytest.mark.parametrize("int8", [False, True])
def test_offsets_past_32_bits(int8):
    """The last sequence of a cache of more than 2^31 elements a side: attended, appended, kept and read back."""
    b, h, d, room, n = 68, 8, 128, 32000, 700
    big = nn.KVCache(b, h, d, room, device="hip", dtype=torch.float16, quantized=int8)
    one = nn.KVCache(1, h, d, room, device="hip", dtype=torch.float16, quantized=int8)
    assert big.storage[0].numel() > 2 ** 31
    rows = [_rows(1, h, n, d, torch.float16, s) for s in (1, 2)]
    tree = nn.DraftTree(_parents(np.random.default_rng(3), 1, 9)[0])
    new = [_rows(b, x, 9, d, torch.float16, s) for x, s in ((h, 4), (h, 5), (4 * h, 6))]
    outs = []
    with ts.no_grad():
        one.append(*(_wrap(x) for x in rows))
        for x, y in zip(big.storage, one.storage):
            if x is not None:
                x[-1:, :, :n].copy_(y[:, :, :n])
        big.length = n
        for cache, at in ((big, slice(None)), (one, slice(b - 1, b))):
            cache.append_tree(*(_wrap(x[at]) for x in new[:2]), tree, rotary_base=BASE)
            outs.append(nn.cached_attention(_wrap(new[2][at]), cache, tree, rotary_base=BASE)._data)
            cache.keep(n, np.tile([[8, 0, 3]], (cache.batch_size, 1)))
            outs += [x._data for x in cache.get(5)]
    for got, want in zip(outs[:3], outs[3:]):
        assert (got[-1:].double() - want.double()).norm() <= 2.0 ** -10 * want.double().norm()


def test_more_codes_than_a_grid_holds():
    """4.4e9 codes a side, read one by one: rows of 9."""
    h, d, n = 64, 9, 7_600_000
    cache = nn.KVCache(1, h, d, n, device="hip", dtype=torch.float16, quantized=True)
    full = (0, 3, 31, 62, 63)
    for x in cache.storage[:2]:
        for head in full:
            x[0, head].copy_(torch.randint(-127, 128, x[0, head].shape, device="cuda", generator=_gen(head)))
    for x in cache.storage[2:]:
        x[0, 63].copy_(2.0 ** (6 * torch.rand(x[0, 63].shape, device="cuda", generator=_gen(d)) - 14))
    cache.length = n
    print("cached read", h, d, n, flush=True)
    for got, x, s in zip(cache.get(), cache.storage[:2], cache.storage[2:]):
        for head in range(h):
            want = (x[0, head].float() * s[0, head]).half() if head in full else 0
            assert (got._data[0, head] == want).all(), head
