"""Attention through a sliding window with sinks, against float64.

The kernels differ from the causal ones in the tiles that they visit and in the elements
that they mask there, so the bounds are the causal tests': relative 2-norms of 1e-2 in
f16 / bf16 (P and dS round to the type, by 2^-11 and 2^-8 of an element at most) and 2e-5 in f32, and no
element further off than 40 times that of the larger of itself and the root mean square.  A
wrong tile or border is an error of the order of 1 in the rows it concerns, which is why
rows are compared one by one as well (each row's own norm, 10 times the bound).

A query that sees one key has P = 1 and dS = dP - delta = 0: there both are fp32 sums of
the same d products dO V in another order (O is V, unrounded), each off by at most d u of
the products' sizes, u = 2^-24.  So the bound of a dq or dk that is nothing else is 2 d u max|dO V| summed
over d, times max|k| scale (max|q| scale, and the rows that see a key) of each term: `floor`.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("no GPU", allow_module_level=True)

import tensorsmith_hip as ts  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402

BOUND = {torch.float16: 1e-2, torch.bfloat16: 1e-2, torch.float32: 2e-5}


def _wrap(x, grad=False):
    return ts.Tensor(x, device="hip", requires_grad=grad)


def _seen(sq, sk, offset, window, sinks):
    i, j = torch.arange(sq, device="cuda")[:, None] + offset, torch.arange(sk, device="cuda")[None]
    return (j <= i) & ((j > i - window) | (j < sinks))


def _reference(q, k, v, up, seen):
    """out, dq, dk, dv in float64; seen broadcasts to [B, H, Q, K]; rows that see nothing give 0."""
    b, h, sq, d = q.shape
    hkv = k.shape[1]
    rep = h // hkv
    q, up = q.double(), up.double()
    kr, vr = (x.double().repeat_interleave(rep, 1) for x in (k, v))
    x = torch.matmul(q, kr.transpose(-1, -2)) / math.sqrt(d)
    x = x.masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    out = torch.matmul(p, vr)
    dv = torch.matmul(p.transpose(-1, -2), up)
    ds = p * (torch.matmul(up, vr.transpose(-1, -2)) - (up * out).sum(-1, keepdim=True)) / math.sqrt(d)
    dq, dk = torch.matmul(ds, kr), torch.matmul(ds.transpose(-1, -2), q)
    group = lambda g: g.view(b, hkv, rep, *g.shape[2:]).sum(2)  # noqa: E731
    return out, dq, group(dk), group(dv)


def _floor(q, k, v, up, seen):
    d, rep = q.shape[3], q.shape[1] // k.shape[1]
    ds = 2 * d * 2.0 ** -24 * up.double().abs().max() * v.double().abs().max() * d
    scale = 1 / math.sqrt(d)
    rows, keys = seen.sum(-2).max().item() * rep, seen.sum(-1).max().item()
    return {"dq": (ds * keys * k.double().abs().max() * scale).item(),
            "dk": (ds * rows * q.double().abs().max() * scale).item()}


def _close(name, got, want, dtype, floor=0.0):
    bound = BOUND[dtype]
    err, norm = (got.double() - want), want.norm()
    rms = want.square().mean().sqrt()
    if norm == 0:
        assert (err.abs() <= floor).all(), name
        return
    assert err.norm() <= bound * norm, (name, (err.norm() / norm).item())
    assert (err.abs() <= 40 * bound * torch.maximum(rms, want.abs())).all(), name
    rows, sizes = err.norm(dim=-1), want.norm(dim=-1)
    # (a row of small values is a sum of the usual terms: its errors are theirs)
    assert (rows <= 10 * bound * torch.maximum(sizes, sizes.square().mean().sqrt())).all(), name


def _operands(b, h, hkv, sq, sk, d, dv, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + sq + sk)
    make = lambda hh, s, c: torch.randn((b, s, hh, c), generator=gen, device="cuda").to(dtype).permute(0, 2, 1, 3)  # noqa: E731
    return make(h, sq, d), make(hkv, sk, d), make(hkv, sk, dv), make(h, sq, dv)


def _run(q, k, v, up, window, sinks, **kw):
    leaves = [_wrap(x, True) for x in (q, k, v)]
    out = nn.scaled_dot_product_attention(*leaves, is_causal=True, window=window, sinks=sinks, enable_gqa=True, **kw)
    out.backward(_wrap(up))
    return (out._data, *(x._grad for x in leaves))


def _check(q, k, v, up, window, sinks, **kw):
    got = _run(q, k, v, up, window, sinks, **kw)
    seen = _seen(q.shape[2], k.shape[2], kw.get("causal_offset", 0), window, sinks)
    want = _reference(q, k, v, up, seen)
    floor = _floor(q, k, v, up, seen)
    if (seen.sum(-1) <= 1).all():  # nothing but the floor: P is 1 whatever the scores
        want = (want[0], torch.zeros_like(want[1]), torch.zeros_like(want[2]), want[3])
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        _close(name, a, b, q.dtype, floor.get(name, 0.0))


WINDOWS = [(1, 0), (1, 1), (7, 3), (31, 0), (32, 32), (33, 5), (64, 0), (100, 130), (128, 33), (300, 64), (515, 1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_training_matches_float64(window, sinks, d, dtype):
    for b, h, hkv, s in ((1, 2, 1, 517), (2, 3, 3, 200)):
        print("window", window, sinks, d, dtype, s, flush=True)
        _check(*_operands(b, h, hkv, s, s, d, d, dtype), window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("s", [1, 2, 31, 33, 127, 128, 129, 1000])
def test_lengths(s, dtype):
    for window, sinks in ((1, 0), (2, 1), (max(1, s - 1), 2), (max(1, s // 3), 0), (s, 0), (s + 5, 1), (10 ** 12, 3)):
        print("window", s, window, sinks, dtype, flush=True)
        _check(*_operands(1, 4, 2, s, s, 64, 64, dtype), window, sinks)


@pytest.mark.parametrize("d,dv", [(128, 64), (64, 128)])
def test_values_of_other_dims(d, dv):
    _check(*_operands(2, 4, 2, 300, 300, d, dv, torch.float16), 70, 9)


def test_long_sequences_cut_the_sinks_blocks():
    """Many parts of the sinks' rows, and sinks of more than one key block."""
    for s, window, sinks, d in ((4100, 40, 4, 128), (3001, 200, 140, 64), (2500, 1, 300, 32)):
        print("window", s, window, sinks, d, flush=True)
        q, k, v, up = _operands(1, 2, 1, s, s, d, d, torch.bfloat16)
        _check(q, k, v, up, window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_queries_behind_a_prefix(dtype):
    for sq, sk, offset, window, sinks in ((5, 700, 695, 64, 4), (130, 700, 570, 200, 0), (130, 300, 400, 50, 33),
                                          (64, 100, 900, 30, 2), (64, 100, 900, 30, 0)):
        print("window", sq, sk, offset, window, sinks, dtype, flush=True)
        _check(*_operands(1, 4, 2, sq, sk, 64, 64, dtype), window, sinks, causal_offset=offset)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padding_that_leaves_rows_empty(dtype):
    q, k, v, up = _operands(3, 4, 2, 300, 300, 64, 64, dtype)
    keep = torch.zeros((3, 1, 1, 300), dtype=torch.bool, device="cuda")
    keep[0, ..., :300], keep[1, ..., :41], keep[2, ..., 20:200:3] = True, True, True
    for window, sinks in ((50, 0), (50, 4), (3, 1)):
        got = _run(q, k, v, up, window, sinks, attn_mask=_wrap(keep))
        want = _reference(q, k, v, up, _seen(300, 300, 0, window, sinks) & keep)
        for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
            _close(name, a, b, dtype)
        if sinks == 0:
            assert (got[0][1, :, 41 + window:] == 0).all()  # those rows see no key


@pytest.mark.parametrize("kind", ["bool", "bias", "half"])
def test_masks_take_the_window_in(kind):
    q, k, v, up = _operands(2, 4, 2, 190, 190, 64, 64, torch.float16)
    gen = torch.Generator(device="cuda").manual_seed(3)
    keep = torch.rand((1, 4, 190, 190), generator=gen, device="cuda") < 0.7
    bias = torch.randn((1, 4, 190, 190), generator=gen, device="cuda")
    mask = keep if kind == "bool" else bias if kind == "bias" else bias.half()
    got = _run(q, k, v, up, 40, 3, attn_mask=_wrap(mask))
    seen = _seen(190, 190, 0, 40, 3)
    if kind == "bool":
        want = _reference(q, k, v, up, seen & keep)[0]
    else:
        x = torch.matmul(q.double(), k.double().repeat_interleave(2, 1).transpose(-1, -2)) / 8 + mask.double()
        want = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v.double().repeat_interleave(2, 1)
    _close("out", got[0], want, torch.float16)


def test_other_types_and_dims_go_by_a_mask():
    for dtype, d in ((torch.float64, 64), (torch.float32, 48), (torch.float16, 40)):
        q, k, v, up = _operands(1, 4, 2, 150, 150, d, d, dtype)
        got = _run(q, k, v, up, 30, 5)
        want = _reference(q, k, v, up, _seen(150, 150, 0, 30, 5))
        for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
            _close(name, a, b, torch.float16 if dtype == torch.float16 else torch.float32)


def test_dropout_keeps_to_the_window():
    q, k, _, _ = _operands(1, 2, 2, 128, 128, 64, 64, torch.float16)
    v = torch.eye(128, 64, device="cuda", dtype=torch.float16)[None, None].expand(1, 2, 128, 64)
    ts.seed(5)
    with ts.no_grad():
        out = nn.scaled_dot_product_attention(_wrap(q), _wrap(k), _wrap(v), dropout_p=0.25, is_causal=True, window=9)
    assert (out._data[..., ~_seen(128, 64, 0, 9, 0)] == 0).all() and (out._data != 0).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_layer_with_rope(dtype):
    """The layer's window, rotations folded in, equals the same layer given the window as a mask."""
    name = str(dtype).split(".")[-1]
    layers = []
    for window, sinks in ((48, 5), (None, 0)):
        ts.seed(1)
        layers.append(nn.MultiHeadAttention(256, 4, num_kv_heads=2, device="hip", window=window, sinks=sinks))
        layers[-1].to(dtype=name)
    x = torch.randn((2, 330, 256), device="cuda").to(dtype)
    up = torch.randn((2, 330, 256), device="cuda").to(dtype)
    mask = _wrap(_seen(330, 330, 0, 48, 5)[None, None])
    results = []
    for layer, kw in ((layers[0], {}), (layers[1], {"attn_mask": mask})):
        leaf = _wrap(x, True)
        out = layer(leaf, **kw)
        out.backward(_wrap(up))
        results.append([out._data, leaf._grad, *(p._grad for p in layer.parameters())])
    for a, b in zip(*results):
        assert (a.double() - b.double()).norm() <= 2 * BOUND[dtype] * b.double().norm()


def test_gradients_match_differences():
    q, k, v, up = _operands(1, 2, 1, 40, 40, 32, 32, torch.float32)
    grads = _run(q, k, v, up, 6, 2)[1:]
    seen = _seen(40, 40, 0, 6, 2)
    value = lambda *x: (_reference(*x, up, seen)[0] * up.double()).sum().item()  # noqa: E731
    for n, (t, g) in enumerate(zip((q, k, v), grads)):
        for at in ((0, 0, 0, 3), (0, 0, 1, 7), (0, 0, 17, 0), (0, 0, 39, 31)):
            x = [y.double() for y in (q, k, v)]
            step = torch.zeros_like(x[n])
            step[at] = 1e-4
            up_, down = list(x), list(x)
            up_[n], down[n] = x[n] + step, x[n] - step
            slope = (value(*up_) - value(*down)) / 2e-4
            assert abs(g[at].item() - slope) <= 2e-5 * (abs(slope) + g.double().square().mean().sqrt().item())


def test_the_same_every_time_and_in_a_graph():
    q, k, v, up = _operands(2, 4, 2, 700, 700, 128, 128, torch.bfloat16)
    first = _run(q, k, v, up, 90, 4)
    for a, b in zip(first, _run(q, k, v, up, 90, 4)):
        assert torch.equal(a, b)
    held = [_wrap(x, True) for x in (q, k, v)]
    alive = nn.scaled_dot_product_attention(*held, is_causal=True, window=90, sinks=4, enable_gqa=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(q, k, v, up, 90, 4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(q, k, v, up, 90, 4)
    for seed in range(3):
        new = _operands(2, 4, 2, 700, 700, 128, 128, torch.bfloat16, seed=seed + 1)
        for a, b in zip((q, k, v, up), new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, _run(*new, 90, 4)):
            assert torch.equal(a, b)
    alive.backward(_wrap(up))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,d", [(2, 64), (3, 128), (5, 32), (7, 64), (20, 128)])
def test_gradients_of_few_keys_lose_nothing_to_the_rounded_output(window, d, dtype):
    """Where a row sees few keys, dP - delta is small beside delta: delta comes from the output as it was before
    its rounding.  What is left are dS's rounding and the result's own, each of at most u = eps / 2 of a value,
    0.42 u in the root mean square (uniform over the last place, values over a binade): together 0.6 u of the norm of
    many independent values, and 0.72 u with a fifth to spare."""
    q, k, v, up = (torch.randn((2, 4, 600, d), generator=torch.Generator(device="cuda").manual_seed(s), device="cuda")
                   .to(dtype) for s in range(4))
    leaves = [_wrap(x, True) for x in (q, k, v)]
    out = nn.scaled_dot_product_attention(*leaves, is_causal=True, window=window)
    out.backward(_wrap(up))
    want = _reference(q, k, v, up, _seen(600, 600, 0, window, 0))
    for name, leaf, exact in zip("qk", leaves, want[1:3]):
        off = ((leaf._grad.double() - exact).norm() / exact.norm()).item()
        assert off <= 0.72 * torch.finfo(dtype).eps / 2, (name, off)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("sinks", [130, 300, 1000])
def test_sinks_of_many_blocks_and_heads(sinks, dtype):
    """Blocks enough to fill the chip are cut into fewer parts, down to none."""
    print("window", sinks, dtype, flush=True)
    _check(*_operands(32, 8, 8, 1100, 1100, 32, 32, dtype), 5, sinks)
