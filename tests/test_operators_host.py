"""Windowed attention, drafted trees over a cache and token log probabilities on the host:
what they refuse, what a refusal leaves as it was, and where and with what they launch."""

from __future__ import annotations

import copy
import ctypes
import pickle
import weakref

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tensorsmith_hip as ts  # noqa: E402
from tensorsmith_hip import _lib, nn  # noqa: E402
from tensorsmith_hip.nn import functional as F  # noqa: E402
from test_host_launches import lib  # noqa: E402,F401  (CPU tensors as device ones, the library as a stub)

INVALID, UNSUPPORTED = 1, 2


def _draw(*shape, dev="hip:0", dtype=torch.float16, grad=False):
    return ts.Tensor(torch.randn(shape).to(dtype), device=dev, requires_grad=grad)


def _ints(values, dev="hip:0", dtype=torch.int64):
    return ts.Tensor(torch.tensor(values, dtype=dtype), device=dev)


def _cache(n=10, room=20, heads=2, d=64, dtype="float16", quantized=False, dev="hip:0", batch=2):
    cache = nn.KVCache(batch, heads, d, room, device=dev, dtype=dtype, quantized=quantized)
    cache.length = n
    return cache


@pytest.mark.parametrize("index", [0, 1])
def test_launches_on_the_tensors_device(lib, index):
    dev = f"hip:{index}"
    got = F.token_log_probs(_draw(3, 5, 40, dev=dev, grad=True), _ints([[1] * 5] * 3, dev), 4)
    assert got.top_indices.shape == (3, 5, 4) and got.entropy.shape == (3, 5)
    (got.log_probs + got.entropy).sum().backward()
    q, k, v = (_draw(2, h, 50, 64, dev=dev, grad=True) for h in (4, 2, 2))
    out = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True, window=8, sinks=2)
    out.backward(_draw(2, 4, 50, 64, dev=dev))
    tree = nn.DraftTree([-1, 0, 0], device=dev)
    cache = _cache(dev=dev)
    with ts.no_grad():
        cache.append_tree(_draw(2, 2, 3, 64, dev=dev), _draw(2, 2, 3, 64, dev=dev), tree, rotary_base=10000.0)
        nn.cached_attention(_draw(2, 4, 3, 64, dev=dev), cache, tree, rotary_base=10000.0)
        cache.keep(10, [[0, 2], [1, 0]])
    assert cache.length == 12
    assert {name for name, _, _ in lib.calls} >= {
        "tsattn_token_probs", "tsattn_token_probs_backward", "tsattn_window_forward", "tsattn_window_backward",
        "tsattn_draft_tree", "tsattn_draft_append", "tsattn_cached_attend", "tsattn_cache_keep"}
    for name, current, stream in lib.calls:
        if name.startswith(("tsattn_token", "tsattn_window", "tsattn_draft", "tsattn_cache")):
            assert (current, getattr(stream, "value", stream)) == (index, 0x100 + index), name
    assert lib.current == 0


def test_token_log_probs_refuses(lib):
    z, y = _draw(4, 9), _ints([0, 1, 2, 3])
    for bad, error in (((_draw(4, 0), y), ValueError), ((_draw(4, 9, 2), y), ValueError), ((z, _ints([0])), ValueError),
                       ((z, _draw(4)), TypeError), ((_ints([[1] * 9] * 4), y), ValueError),
                       ((z, _ints([0, 1, 2, 3], "hip:1")), ValueError), ((_draw(4, 9, dtype=torch.float64), y), TypeError),
                       ((z, y, -1), ValueError), ((z, y, 10), ValueError), ((z, y, True), ValueError),
                       ((z, y, 2.0), ValueError), ((_draw(4, 100), y, 65), ValueError)):
        with pytest.raises(error):
            F.token_log_probs(*bad)
    with pytest.raises(TypeError):
        F.token_log_probs(z, y, ignore_index=0.5)
    with pytest.raises(ValueError, match="require gradients"):
        F.token_log_probs(z, ts.Tensor(torch.zeros(4), device="hip:0", requires_grad=True))
    assert not lib.calls
    F.token_log_probs(z, y, ignore_index=np.int64(-7))
    assert lib.args["tsattn_token_probs"][7] == -7


@pytest.mark.parametrize("kind", [int, np.int32, np.int64, np.uint8])
def test_top_k_of_any_integer_type(lib, kind):
    got = F.token_log_probs(_draw(4, 9), _ints([0, 1, 2, 3]), kind(3))
    assert got.top_log_probs.shape == got.top_indices.shape == (4, 3)
    assert lib.args["tsattn_token_probs"][8] == 3 and type(lib.args["tsattn_token_probs"][8]) is int
    with pytest.raises(ValueError, match="top_k"):
        F.token_log_probs(_draw(4, 9), _ints([0, 1, 2, 3]), kind(10))


def test_no_rows_launch_nothing(lib):
    z = _draw(0, 3, 9, grad=True)
    got = F.token_log_probs(z, _ints(np.zeros((0, 3), np.int64).tolist()).reshape(0, 3), 2)
    assert got.log_probs.shape == (0, 3) and got.top_log_probs.shape == (0, 3, 2)
    got.log_probs.sum().backward()
    assert z.grad.shape == (0, 3, 9)
    assert not [name for name, _, _ in lib.calls if "token_probs" in name]


def test_windows_are_checked(lib):
    q = _draw(1, 2, 6, 64)
    for kw, error in (({"window": 0}, "window"), ({"window": -3}, "window"), ({"window": True}, "window"),
                      ({"window": 2.0}, "window"), ({"sinks": 2}, "sinks"), ({"window": 3, "sinks": -1}, "sinks"),
                      ({"window": 3, "sinks": 1.5}, "sinks"), ({"window": 3, "is_causal": False}, "causal")):
        with pytest.raises(ValueError, match=error):
            F.scaled_dot_product_attention(q, q, q, **{"is_causal": True, **kw})
        if "is_causal" in kw:
            continue
        with pytest.raises(ValueError, match=error), ts.no_grad():
            nn.cached_attention(_draw(2, 2, 1, 64), _cache(), **kw)
        with pytest.raises(ValueError, match=error):
            nn.MultiHeadAttention(128, 2, device="hip:0", **kw)
        with pytest.raises(ValueError, match=error):
            nn.TransformerConfig(vocab_size=10, dim=128, num_heads=2, num_layers=1, max_seq_len=16,
                                 **{"attention_" + name: x for name, x in kw.items()})
    layer = nn.MultiHeadAttention(128, 2, window=4, device="hip:0")
    with pytest.raises(ValueError, match="causal"):
        layer(_draw(1, 6, 128, dtype=torch.float32), is_causal=False)
    assert not lib.calls


def test_layers_pickled_before_windows_run(lib):
    """They hold neither window nor sinks."""
    layer = nn.MultiHeadAttention(128, 2, rotary=False, device="hip:0")
    del layer.__dict__["window"], layer.__dict__["sinks"]
    layer = pickle.loads(pickle.dumps(layer)).eval()
    assert layer(_draw(1, 3, 128, dtype=torch.float32)).shape == (1, 3, 128)
    with ts.no_grad():
        assert layer(_draw(1, 3, 128, dtype=torch.float32), cache=layer.new_cache(1, 8)).shape == (1, 3, 128)
    assert not [name for name, _, _ in lib.calls if "window" in name]


def test_windows_as_the_library_takes_them(lib):
    """Any integers, no larger than they can count; a window over everything is none."""
    q = _draw(1, 2, 60, 64)
    F.scaled_dot_product_attention(q, q, q, is_causal=True, window=np.int32(8), sinks=2**40)
    assert lib.args["tsattn_window_forward"][1:3] == (8, 60)
    assert all(type(x) is int for x in lib.args["tsattn_window_forward"][1:3])
    lib.calls.clear()
    F.scaled_dot_product_attention(q, q, q, is_causal=True, window=60, sinks=3)
    assert not [name for name, _, _ in lib.calls if "window" in name]
    with ts.no_grad():
        nn.cached_attention(_draw(2, 2, 1, 64), _cache(), window=np.int64(5), sinks=np.int64(2**33))
        desc = lib.args["tsattn_cached_attend"][0]
        assert (desc.window, desc.sinks, desc.keys, desc.len) == (5, 10, 10, 1)
        nn.cached_attention(_draw(2, 2, 1, 64), _cache(), window=2**40, sinks=1)
        desc = lib.args["tsattn_cached_attend"][0]
        assert (desc.window, desc.sinks) == (0, 0)


def test_trees_are_checked(lib):
    for bad in ([0], [-2], [-1, 1], [-1, -1, 3], [2**32 - 1], [-2**40], [], [[]], [[[-1]]], [-1] * 257):
        with pytest.raises(ValueError):
            nn.DraftTree(bad, device="hip:0")
    for bad in ([0.5], [-1.0], [True], ts.Tensor(torch.zeros(3), device="hip:0")):
        with pytest.raises(TypeError):
            nn.DraftTree(bad, device="hip:0")
    with pytest.raises(ValueError, match="device"):
        nn.DraftTree(_ints([-1, 0], "hip:1"), device="hip:0")
    assert not lib.calls
    assert nn.DraftTree([-1] * 256, device="hip:0").tokens == 256
    seen = []
    lib.__dict__["tsattn_draft_tree"] = lambda trees, n, parents, *rest: seen.append(
        [ctypes.c_int32.from_address(parents + 4 * i).value for i in range(trees * n)]) or 0
    # values on the device are not waited for; none wraps round to an earlier token
    nn.DraftTree(_ints([-1, 2**32, -2**32, 2**33 + 1, 3], "hip:1"))
    assert seen[0][0] == -1 and seen[0][4] == 3
    assert all(not 0 <= p < t for t, p in enumerate(seen[0][:4]))


def test_drafted_rows_are_checked_before_the_cache_takes_them(lib):
    tree, rows = nn.DraftTree([-1, 0, 0], device="hip:0"), _draw(2, 2, 3, 64)
    lib.calls.clear()
    cache = _cache()
    with ts.no_grad():
        for args, kw, error in (((_draw(2, 2, 4, 64), _draw(2, 2, 4, 64), tree), {}, "tree"),
                                ((rows, rows, nn.DraftTree([[-1, 0, 0]] * 3, device="hip:0")), {}, "tree"),
                                ((rows, rows, nn.DraftTree([-1, 0, 0], device="hip:1")), {}, "device"),
                                ((rows, rows, tree), {"rotary_base": -1.0}, "RoPE"),
                                ((rows, rows, tree), {"rotary_base": float("inf")}, "RoPE"),
                                ((rows, _draw(2, 2, 2, 64), tree), {}, "shape")):
            lib.calls.clear()
            with pytest.raises(ValueError, match=error):
                cache.append_tree(*args, **kw)
            assert cache.length == 10 and not [name for name, _, _ in lib.calls if "append" in name]
        full = _cache(n=18)
        with pytest.raises(ValueError, match="capacity"):
            full.append_tree(rows, rows, tree)
    with pytest.raises(RuntimeError, match="inference"):
        cache.append_tree(_draw(2, 2, 3, 64, grad=True), rows, tree)


def test_a_layer_refuses_drafts_before_its_cache_takes_them(lib):
    layer = nn.MultiHeadAttention(128, 2, window=2, device="hip:0").eval()
    tree, cache = nn.DraftTree([-1, 0, 0], device="hip:0"), layer.new_cache(2, 20)
    x = _draw(2, 3, 128, dtype=torch.float32)
    with ts.no_grad():
        with pytest.raises(ValueError, match="window must hold"):
            layer(x, cache=cache, tree=tree)
        for kw in ({"cache": None}, {"cache": cache, "is_causal": False},
                   {"cache": cache, "attn_mask": ts.Tensor(torch.ones(3, 3, dtype=torch.bool), device="hip:0")}):
            with pytest.raises(ValueError):
                layer(x, tree=tree, **kw)
    assert cache.length == 0
    model = nn.TransformerLM(nn.TransformerConfig(vocab_size=10, dim=64, num_heads=2, num_layers=2, max_seq_len=16,
                                                  attention_window=2), device="hip:0").eval()
    caches = model.new_cache(1)
    with ts.no_grad():
        with pytest.raises(ValueError, match="window must hold"):
            model(_ints([[1, 2, 3]]), caches=caches, tree=tree)
        with pytest.raises(ValueError, match="tree"):
            model(_ints([[1, 2]]), caches=caches, tree=tree)
        with pytest.raises(ValueError, match="KVCache"):
            model(_ints([[1, 2, 3]]), tree=tree)
    assert [c.length for c in caches] == [0, 0]


def test_cached_attention_refuses(lib):
    cache, q = _cache(), _draw(2, 4, 3, 64)
    tree = nn.DraftTree([-1, 0, 0], device="hip:0")
    lib.calls.clear()
    with ts.no_grad():
        with pytest.raises(TypeError):
            nn.cached_attention(q, (q, q))
        with pytest.raises(TypeError):
            nn.cached_attention(_draw(2, 4, 3, 64, dtype=torch.float32), cache)
        for bad, kw in ((_draw(2, 4, 64), {}), (_draw(1, 4, 3, 64), {}), (_draw(2, 3, 3, 64), {}),
                        (_draw(2, 4, 3, 32), {}), (_draw(2, 0, 3, 64), {}), (_draw(2, 4, 0, 64), {}),
                        (_draw(2, 4, 11, 64), {}), (_draw(2, 4, 3, 64, dev="hip:1"), {}),
                        (q, {"scale": float("nan")}), (q, {"rotary_base": 0.0}),
                        (q, {"tree": tree, "window": 2}), (_draw(2, 4, 2, 64), {"tree": tree}),
                        (q, {"tree": nn.DraftTree([[-1, 0, 0]] * 3, device="hip:0")})):
            with pytest.raises(ValueError):
                nn.cached_attention(bad, cache, **kw)
    with pytest.raises(RuntimeError, match="inference"):
        nn.cached_attention(_draw(2, 4, 3, 64, grad=True), cache)
    assert not [name for name, _, _ in lib.calls if "attend" in name]


def test_kept_rows_are_checked(lib):
    cache = _cache()
    for first, index, error in ((-1, [[0], [0]], ValueError), (11, [[0], [0]], ValueError), (1.5, [[0], [0]], TypeError),
                                (7, [[3], [0]], ValueError), (7, [[-1], [0]], ValueError), (7, [0, 1], ValueError),
                                (7, [[0]], ValueError), (7, [[0, 1, 2, 0]] * 2, ValueError),
                                (7, [[0.0], [1.0]], TypeError), (7, _ints([[0], [0]], "hip:1"), ValueError)):
        with pytest.raises(error):
            cache.keep(first, index)
        assert cache.length == 10 and not lib.calls
    cache.keep(np.int64(7), np.zeros((2, 0), np.int64))
    assert cache.length == 7 and type(cache.length) is int and not lib.calls
    cache.keep(2, _ints([[4, 4], [0, 3]], dtype=torch.int32))
    args = lib.args["tsattn_cache_keep"]
    assert cache.length == 4 and args[:5] == (2, 2, 2, 2, 5) and args[6:10] == (4, 2, 64, 64)


def test_the_last_rows_of_a_cache(lib):
    cache = nn.KVCache(2, 2, 8, 12, device="hip:0", dtype="float32")
    cache.storage[0][:, :, :9], cache.storage[1][:, :, :9] = torch.randn(2, 2, 9, 8), torch.randn(2, 2, 9, 8)
    cache.length = 9
    whole = cache.get()
    for last in (0, 1, 4, 9, np.int32(3)):
        for part, all_ in zip(cache.get(last), whole):
            assert torch.equal(part._data, all_._data[:, :, 9 - last:])
    for bad in (-1, 10):
        with pytest.raises(ValueError):
            cache.get(bad)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("again", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_a_cache_in_use_can_be_copied(lib, again, quantized):
    cache = _cache(quantized=quantized)
    tree = nn.DraftTree([-1, 0], device="hip:0")
    with ts.no_grad():
        cache.get()
        cache.append_tree(_draw(2, 2, 2, 64), _draw(2, 2, 2, 64), tree)
        nn.cached_attention(_draw(2, 2, 2, 64), cache, tree)
        cache.keep(10, [[1], [0]])
        other = again(cache)
        assert other.length == cache.length == 11 and other.device == cache.device
        assert all(torch.equal(a, b) and a.data_ptr() != b.data_ptr()
                   for a, b in zip(cache.storage, other.storage) if a is not None)
        nn.cached_attention(_draw(2, 2, 2, 64), other)
        assert lib.args["tsattn_cached_attend"][2].data == other._keys.data_ptr()
        shared = copy.copy(cache)  # (another cache over the same arrays)
        assert shared._keys is cache._keys and len(shared) == 11


@pytest.mark.parametrize("quantized", [False, True])
def test_a_reordered_cache_lets_its_old_arrays_go(lib, quantized):
    cache = _cache(quantized=quantized)
    with ts.no_grad():
        nn.cached_attention(_draw(2, 2, 1, 64), cache)
        old = [weakref.ref(x) for x in cache.storage if x is not None]
        cache.reorder([1, 0])
        assert all(x() is None for x in old)
        nn.cached_attention(_draw(2, 2, 1, 64), cache)
        assert lib.args["tsattn_cached_attend"][2].data == cache._keys.data_ptr()


def test_codes_are_read_on_the_caches_device(lib):
    cache = nn.KVCache(2, 3, 8, 12, device="hip:1", dtype="float16", quantized=True, value_dim=5)
    assert [x.shape for x in cache.get()] == [(2, 3, 0, 8), (2, 3, 0, 5)] and not lib.calls
    cache.length = 9
    assert [x.shape for x in cache.get(4)] == [(2, 3, 4, 8), (2, 3, 4, 5)]
    name, current, stream = lib.calls[-1]
    assert (name, current, getattr(stream, "value", stream)) == ("tsattn_kv_read_int8", 1, 0x101)
    args = lib.args[name]
    assert args[:7] == (_lib.F16, 2, 3, 5, 4, 8, 5)
    assert [x.data for x in args[7:11]] == [x.data_ptr() for x in cache.storage]
    lib.__dict__.update(tsattn_kv_read_int8=lambda *a: UNSUPPORTED, tsattn_last_error=lambda: b"unsupported")
    for x in cache.storage[:2]:
        x[:] = torch.randint(-127, 128, x.shape).to(torch.int8)
    for x in cache.storage[2:]:
        x[:] = torch.rand(x.shape)
    for got, codes, scales in zip(cache.get(4), cache.storage[:2], cache.storage[2:]):
        assert torch.equal(got._data, (codes[:, :, 5:9].float() * scales[:, :, 5:9]).half())


# -- the library itself ------------------------------------------------------------------

def _view(address=0x1000, stride=(4096, 1024, 64, 1)):
    v = _lib.View()
    v.data = address
    v.stride[:] = stride
    return v


def _problem(**kw):
    p = _lib.Problem(dtype=_lib.F16, batch=1, heads_q=2, heads_kv=2, len_q=16, len_kv=16, dim_qk=64, dim_v=64,
                     is_causal=1, scale=0.125, mask_kind=_lib.MASK_NONE)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def _code(result):
    return abs(result)


def test_the_library_refuses_windows():
    real, v = _lib.load(), _view()
    for window, sinks, p in ((0, 0, {}), (-1, 0, {}), (4, -1, {}), (4, 0, {"is_causal": 0}), (4, 0, {"len_q": 0})):
        rc = real.tsattn_window_forward(ctypes.byref(_problem(**p)), window, sinks, None, v, v, v, v, None, None, None)
        assert _code(rc) == INVALID, (window, sinks, p)
        assert real.tsattn_window_backward_workspace(ctypes.byref(_problem(**p)), window, sinks, 0) == 0
    for p in ({"dim_qk": 48, "dim_v": 48}, {"dropout_p": 0.5}):
        rc = real.tsattn_window_forward(ctypes.byref(_problem(**p)), 4, 0, None, v, v, v, v, None, None, None)
        assert _code(rc) == UNSUPPORTED, p
    # (views that are not 16-byte aligned have no windowed kernel)
    rc = real.tsattn_window_forward(ctypes.byref(_problem()), 4, 0, None, _view(0x1002), v, v, v, None, None, None)
    assert _code(rc) == UNSUPPORTED
    for low, kw in ((0x1008, {}), (0x1000, {"dtype": _lib.F32})):  # (aligned, and of 16 bits)
        rc = real.tsattn_window_forward(ctypes.byref(_problem(**kw)), 4, 0, None, v, v, v, v, None, low, None)
        assert _code(rc) == INVALID
    need = real.tsattn_window_backward_workspace(ctypes.byref(_problem(len_q=600, len_kv=600)), 4, 1, 0)
    assert need > 0
    rc = real.tsattn_window_backward(ctypes.byref(_problem(len_q=600, len_kv=600)), 4, 1, None, v, v, v, v, v, 0x1000,
                                     None, v, v, v, 0x1000, need - 1, None)
    assert _code(rc) == INVALID


@pytest.mark.parametrize("dtype,d", [(_lib.F16, 64), (_lib.BF16, 128), (_lib.F32, 128), (_lib.F32, 32)])
def test_the_scratch_of_sinks_is_bounded(dtype, d):
    """At most 256 MiB of partial sums (8 workgroups a CU, each 128 keys of 128 channels), whatever the sinks."""
    real = _lib.load()
    for batch, heads, s, window, sinks in ((8, 8, 32768, 512, 4096), (4, 8, 32768, 128, 4096), (1, 8, 32768, 512, 4096),
                                           (1, 1, 1 << 20, 1, 1 << 19), (64, 8, 8192, 64, 4), (2, 4, 8192, 1024, 4)):
        p = _problem(dtype=dtype, batch=batch, heads_q=heads, heads_kv=heads, len_q=s, len_kv=s, dim_qk=d, dim_v=d)
        need = real.tsattn_window_backward_workspace(ctypes.byref(p), window, sinks, 0)
        rows = real.tsattn_window_backward_workspace(ctypes.byref(p), window, 0, 0)
        assert 0 < rows <= need <= rows + (256 << 20) + 256, (batch, heads, s, window, sinks)


def _cached(**kw):
    d = _lib.Cached(_lib.F16, 2, 4, 2, 64, 3, 10, 0, 0.125, 0, 0, 0, None, None, None, None)
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def test_the_library_refuses_cached_problems():
    real, v = _lib.load(), _view()
    attend = lambda d, q=v, k=v, ks=None, vs=None, ws=None, n=0: _code(  # noqa: E731
        real.tsattn_cached_attend(d, q, k, v, ks, vs, v, ws, n, None))
    for kw in ({"len": 0}, {"len": 11}, {"batch": 0}, {"heads_q": 3}, {"scale": float("nan")}, {"window": -1},
               {"sinks": 1}, {"words": 0x1000}, {"words": 0x1000, "depths": 0x1000, "trees": 3},
               {"words": 0x1000, "depths": 0x1000, "trees": 1, "window": 2}, {"cos": 0x1000}, {"dtype": 99}):
        assert attend(_cached(**kw)) == INVALID, kw
        assert real.tsattn_cached_attend_workspace(_cached(**kw)) == 0
    for kw in ({"dim": 48}, {"dim": 512}, {"dtype": _lib.F64}, {"dtype": _lib.F32, "dim": 256},
               {"dtype": _lib.F32, "quantized": 1}, {"len": 300, "keys": 300}, {"scale": 0.0}, {"scale": -1.0},
               {"cos": 0x1004, "sin": 0x1000}):
        assert attend(_cached(**kw)) == UNSUPPORTED, kw
    assert attend(_cached(), q=_view(0x1002)) == UNSUPPORTED
    assert attend(_cached(), k=_view(stride=(4096, 1024, 36, 1))) == UNSUPPORTED
    assert attend(_cached(keys=1 << 20), k=_view(stride=(4096, 1024, 2048, 1))) == UNSUPPORTED
    long = _cached(keys=100000)
    need = real.tsattn_cached_attend_workspace(long)
    assert need > 0 and attend(long) == INVALID and attend(long, ws=0x1000, n=need - 1) == INVALID
    assert attend(long, ws=0x1004, n=need) == INVALID
    # codes need scales, a value a row and not one for all of them
    codes = _cached(quantized=1)
    assert attend(codes) == INVALID
    scales = _view(stride=(64, 32, 1, 1))
    assert attend(codes, ks=scales) == INVALID
    assert attend(codes, ks=scales, vs=_view(stride=(64, 32, 0, 1))) == UNSUPPORTED
    assert attend(codes, ks=_view(0x1002, (64, 32, 1, 1)), vs=scales) == UNSUPPORTED


def test_the_library_refuses_trees_and_kept_rows():
    real, v = _lib.load(), _view()
    tree = lambda trees, n, p=0x1000: _code(real.tsattn_draft_tree(trees, n, p, 0x1000, 0x1000, None))  # noqa: E731
    assert (tree(0, 3), tree(1, 0), tree(1, 257), tree(1, 3, None)) == (INVALID, INVALID, UNSUPPORTED, INVALID)
    keep = lambda n=2, first=3, limit=4, index=0x1000, ib=8, eb=2, ks=None: _code(  # noqa: E731
        real.tsattn_cache_keep(2, 2, n, first, limit, index, ib, eb, 64, 64, v, v, ks, None, None))
    assert [keep(n=0), keep(n=5), keep(first=-1), keep(index=None), keep(ib=2), keep(eb=3), keep(ks=v)] == [INVALID] * 7
    assert keep(n=257, limit=300) == UNSUPPORTED
    append = lambda depths=0x1000, trees=1, n=3, cos=None: _code(real.tsattn_draft_append(  # noqa: E731
        _lib.F16, 2, 2, n, 64, v, v, v, v, None, None, cos, None, 5, depths, trees, None))
    assert [append(depths=None), append(trees=3), append(cos=0x1000)] == [INVALID] * 3
    assert append(n=257) == UNSUPPORTED


def test_more_workgroups_than_a_grid_holds_are_refused():
    """From 2^24 workgroups of 256 on a grid wraps round without an error."""
    real, v = _lib.load(), _view()
    for kw in ({"batch": 1 << 23}, {"batch": 1 << 16, "heads_q": 1 << 8}, {"batch": 1 << 30, "heads_q": 1 << 20},
               {"dtype": _lib.F32, "batch": 1 << 20, "len_q": 4096, "len_kv": 4096}):
        args = (ctypes.byref(_problem(heads_kv=1, **kw)), 4, 1, None, v, v, v, v)
        assert _code(real.tsattn_window_forward(*args, None, None, None)) == INVALID, kw
        assert _code(real.tsattn_window_backward(*args, v, 0x1000, None, v, v, v, 0x1000, 1 << 62, None)) == INVALID, kw
    for kw in ({"batch": 1 << 23}, {"batch": 1 << 16, "heads_q": 1 << 8, "heads_kv": 1 << 8},
               {"batch": 1 << 30, "heads_q": 1 << 20, "heads_kv": 1 << 20},
               {"batch": 1 << 12, "heads_q": 1 << 7, "heads_kv": 1, "len": 256, "keys": 256}):
        rc = real.tsattn_cached_attend(_cached(**kw), v, v, v, None, None, v, 0x1000, 1 << 62, None)
        assert _code(rc) == INVALID, kw
    assert _code(real.tsattn_draft_tree(1 << 24, 3, 0x1000, 0x1000, 0x1000, None)) == INVALID
    for b, h in ((1 << 23, 1), (1 << 16, 1 << 8), (1 << 30, 1 << 30)):
        rc = real.tsattn_cache_keep(b, h, 2, 3, 4, 0x1000, 8, 2, 64, 64, v, v, None, None, None)
        assert _code(rc) == INVALID, (b, h)
        rc = real.tsattn_draft_append(_lib.F16, b, h, 9, 64, v, v, v, v, None, None, None, None, 5, 0x1000, 1, None)
        assert _code(rc) == INVALID, (b, h)


def test_the_library_refuses_token_probabilities():
    real = _lib.load()

    def probs(dtype=_lib.F16, rows=4, vocab=9, logits=0x1000, stride=9, tokens=0x1000, tb=8, top=0, out=0x1000, ws=None,
              n=0):
        return _code(real.tsattn_token_probs(dtype, rows, vocab, logits, stride, tokens, tb, -100, top, out, 0x1000,
                                             None, None, None, ws, n, None))

    assert [probs(dtype=_lib.F64), probs(rows=0), probs(vocab=0), probs(logits=None), probs(tokens=None), probs(tb=2),
            probs(stride=-1), probs(top=-1), probs(top=10), probs(logits=0x1001), probs(out=None),
            probs(top=3)] == [INVALID] * 12  # (the last: no place for the top tokens)
    assert [probs(vocab=100, top=65), probs(rows=1 << 31), probs(vocab=(1 << 30) + 1)] == [UNSUPPORTED] * 3
    need = real.tsattn_token_probs_workspace(1, 100000, 0)
    assert need > 0 and probs(rows=1, vocab=100000, n=need) == INVALID
    assert probs(rows=1, vocab=100000, ws=0x1000, n=need - 1) == INVALID
    backward = lambda stats=0x1000, entropy=None, ge=None, gt=None, out=0x1000: _code(  # noqa: E731
        real.tsattn_token_probs_backward(_lib.F16, 4, 9, 0x1000, 9, 0x1000, 8, -100, 0, stats, entropy, None, 0x1000,
                                         ge, gt, out, None))
    assert [backward(stats=None), backward(out=None), backward(ge=0x1000), backward(gt=0x1000),
            backward(out=0x1001)] == [INVALID] * 5


def test_the_library_refuses_rows_to_read():
    real, v = _lib.load(), _view()

    def read(dtype=_lib.F16, b=2, h=2, first=3, n=5, dk=8, dv=8, k=v, ks=v, out=0x1000):
        return _code(real.tsattn_kv_read_int8(dtype, b, h, first, n, dk, dv, k, v, ks, v, out, 0x1000, None))

    assert [read(dtype=_lib.BOOL), read(b=0), read(h=0), read(n=0), read(dk=0), read(dv=0), read(k=None), read(ks=None),
            read(out=None), read(first=-1)] == [INVALID] * 10
    assert [read(dtype=_lib.F64), read(n=1 << 28), read(b=1 << 20, h=1 << 12)] == [UNSUPPORTED] * 3
