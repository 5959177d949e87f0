"""Token log probabilities, entropies and top tokens against float64, and their gradients.

Bounds, in units u = 2^-24 of fp32's half step.  With x = z - m and l = sum e^x over V
logits: x is rounded once and scaled once, so e^x is off by (2 |x| + 2) u relative, and
weighted by p the mean of |x| is at most ln V; the sum's own roundings are at most V / 2048
+ 60 in a chain (8 a piece, a lane's pieces, the joins; rescalings telescope to the same
ln V).  So l is off by at most d = (V / 2048 + 64 + 4 ln V) u relative, ln p by d and the
roundings of its two terms, the entropy by d for ln l and 2 d for its second term, at most
ln V.  Of the gradient, p is off by d + (2 |ln p| + 4) u and its factor by 4 u of the sum
of its terms' sizes and gh times the entropy's error; the result is rounded to the
logits' type once.
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
from tensorsmith_hip.nn import functional as F  # noqa: E402

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _wrap(x, grad=False):
    return ts.Tensor(x, device="hip", requires_grad=grad)


def _spread(v):
    return (v / 2048 + 64 + 4 * math.log(v)) * U


def _want(z, y):
    lp = torch.log_softmax(z.double(), -1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    return lp, p, entropy


def _check(z, y, top, got):
    """Every result of rows whose token is in the vocabulary."""
    v = z.shape[-1]
    lp, _, entropy = _want(z, y)
    want = lp.gather(-1, y.long()[..., None])[..., 0]
    d = _spread(v)
    close = lambda a, b, tol: bool((((a.double() - b).abs() <= tol) | (a == b)).all())  # noqa: E731
    assert close(got.log_probs._data, want, d + 3 * U * want.abs().clamp(min=1)), "log_probs"
    assert close(got.entropy._data, entropy, d + 2 * d * math.log(max(v, 3)) + 4 * U * math.log(max(v, 3))), "entropy"
    if top:
        index = torch.sort(z.float(), dim=-1, descending=True, stable=True).indices[..., :top]
        assert torch.equal(got.top_indices._data, index)
        values = lp.gather(-1, index)
        assert close(got.top_log_probs._data, values, d + 3 * U * values.abs().clamp(min=1)), "top"


def _logits(rows, v, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + v)
    z = (2 * torch.randn((rows, v), generator=gen, device="cuda")).to(dtype)
    return z, torch.randint(0, v, (rows,), generator=gen, device="cuda")


SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (9, 63), (2, 65), (777, 100), (6, 1009), (7, 2048), (3, 2049), (1, 16384),
         (2, 16391), (5, 50021), (1, 128001), (70, 9000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", SIZES)
def test_results_match_float64(rows, v, dtype):
    z, y = _logits(rows, v, dtype)
    if v > 8:
        z[:, v // 3: v // 3 + v // 5] = -math.inf
        z[torch.arange(rows), y] = 1.0
    for top in sorted({0, 1, min(5, v), min(64, v)}):
        print("token probs", rows, v, dtype, top, flush=True)
        got = F.token_log_probs(_wrap(z), _wrap(y), top)
        assert got.log_probs.shape == (rows,) and (got.top_indices is None) == (top == 0)
        _check(z, y, top, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("make", ["rising", "falling", "equal", "two", "blocks", "tiny", "huge"])
@pytest.mark.parametrize("v", [257, 2048, 20000, 70001])
def test_orders_that_fill_the_top_lists(make, v, dtype):
    i = torch.arange(v, device="cuda", dtype=torch.float32)
    z = {"rising": i / v * 8, "falling": -i / v * 8, "equal": torch.full_like(i, 0.25), "two": (i % 2),
         "blocks": torch.floor(i / 64) % 7, "tiny": -i.remainder(5) * 1e-5, "huge": 6e4 - 1e2 * i.remainder(11)}[make]
    z = torch.stack((z, z.flip(0))).to(dtype)
    y = torch.tensor([0, v - 1], device="cuda")
    for top in (1, 20, 64):
        print("token probs", make, v, dtype, top, flush=True)
        _check(z, y, top, F.token_log_probs(_wrap(z), _wrap(y), top))


def test_rows_anywhere_in_memory():
    gen = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn((3, 5, 3007), generator=gen, device="cuda").half()
    flat = torch.randn(40000, generator=gen, device="cuda").bfloat16()
    views = [big[:, -1], big[:, 1:4, 5:2905], big[:, :, ::3], big[1:2, 0].expand(4, 3007), big.transpose(0, 1)[2:],
             flat[3:3 + 4 * 5003].view(4, 5003), flat[1:2 + 12001][:12001]]
    for x in views:
        y = torch.randint(0, x.shape[-1], x.shape[:-1], generator=gen, device="cuda", dtype=torch.int32)
        got = F.token_log_probs(_wrap(x), _wrap(y), 9)
        assert got.entropy.shape == tuple(x.shape[:-1]) and got.top_indices.shape == (*x.shape[:-1], 9)
        _check(x, y, 9, got)


def test_padding_and_tokens_outside():
    for v in (100, 40000):
        z, y = _logits(6, v, torch.float32)
        z[0] = math.nan  # (a row that is not read)
        y = torch.tensor([-100, v - 1, v, -1, -(2 ** 40), 2 ** 40 + 1], device="cuda")
        got = F.token_log_probs(_wrap(z), _wrap(y), 3)
        lp, entropy = got.log_probs._data, got.entropy._data
        assert lp[0] == 0 and entropy[0] == 0 and (got.top_log_probs._data[0] == -math.inf).all()
        assert (got.top_indices._data[0] == -1).all()
        assert torch.isnan(lp[2:]).all() and torch.isfinite(entropy[1:]).all() and torch.isfinite(lp[1])
        own = F.token_log_probs(_wrap(z), _wrap(torch.where(y == -100, 7, y)), ignore_index=7)
        assert own.log_probs._data[0] == 0 and torch.equal(own.log_probs._data[1], lp[1])
    none = F.token_log_probs(_wrap(z[:0]), _wrap(y[:0]), 2)
    assert none.log_probs.shape == (0,) and none.top_indices.shape == (0, 2)


@pytest.mark.parametrize("v", [50, 2500, 30000])
def test_rows_without_a_distribution_are_nan(v):
    z, y = _logits(4, v, torch.float32)
    z[0] = -math.inf
    z[1, v // 2] = math.inf
    z[2, v - 1] = math.nan
    got = F.token_log_probs(_wrap(z), _wrap(y), 2)
    assert torch.isnan(got.log_probs._data[:3]).all() and torch.isnan(got.entropy._data[:3]).all()
    assert got.top_indices._data[:3, 0].tolist() == [0, v // 2, v - 1]
    assert got.top_indices._data[0].tolist() == [0, 1]
    _check(z[3:], y[3:], 0, F.token_log_probs(_wrap(z[3:]), _wrap(y[3:])))


def _gradient(z, y, g, gh, gt, index):
    lp, p, entropy = _want(z, y)
    hot = torch.zeros_like(p).scatter_(-1, y[:, None], 1.0)
    finite = torch.where(p > 0, lp, 0.0)
    want = g[:, None] * (hot - p) - gh[:, None] * p * (finite + entropy[:, None])
    size = p * (g.abs() + gh.abs() * (finite.abs() + entropy[:, None].abs()).amax(-1))[:, None]
    if gt is not None:
        want = want - p * gt.sum(-1, keepdim=True)
        want.scatter_add_(1, index, gt)
        size = size + p * gt.abs().sum(-1, keepdim=True)
    v = z.shape[1]
    d = _spread(v)
    tol = size * (d + (2 * finite.abs() + 10) * U)
    tol = tol + p * gh.abs()[:, None] * (d + 2 * d * math.log(max(v, 3)) + 4 * U * math.log(max(v, 3)))
    return want, tol + 4 * U * hot * g.abs()[:, None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v,top", [(1, 1, 1), (3, 7, 0), (9, 130, 4), (5, 1009, 20), (4, 2049, 0), (3, 20001, 7),
                                        (1, 70000, 3), (300, 5003, 2)])
def test_gradients_match_the_formula(rows, v, top, dtype):
    z, y = _logits(rows, v, dtype)
    if v > 8:
        z[:, v // 2:v // 2 + 3] = -math.inf
        y = torch.where((y >= v // 2) & (y < v // 2 + 3), 0, y)
        z[0, y[0]] = z[0].max() + 1  # the token is its row's first alternative
    gen = torch.Generator(device="cuda").manual_seed(v)
    g, gh = (torch.randn(rows, generator=gen, device="cuda") for _ in range(2))
    gt = torch.randn((rows, top), generator=gen, device="cuda") if top else None
    print("token probs vjp", rows, v, top, dtype, flush=True)
    x = _wrap(z, True)
    got = F.token_log_probs(x, _wrap(y), top)
    loss = (got.log_probs * _wrap(g) + got.entropy * _wrap(gh)).sum()
    if top:
        loss = loss + (got.top_log_probs * _wrap(gt)).sum()
    loss.backward()
    want, tol = _gradient(z, y, g.double(), gh.double(), None if gt is None else gt.double(),
                          got.top_indices._data if top else None)
    half = torch.finfo(dtype).eps / 2
    tol = tol + half * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert x._grad.dtype == dtype
    assert ((x._grad.double() - want).abs() <= tol).all()


def test_gradients_of_one_result_and_of_padding():
    z, y = _logits(6, 333, torch.float32)
    y[2] = -100
    for name in ("log_probs", "entropy", "top_log_probs"):
        x = _wrap(z, True)
        got = F.token_log_probs(x, _wrap(y), 3)
        getattr(got, name).sum().backward()
        ones, none = torch.ones(6, device="cuda").double(), torch.zeros(6, device="cuda").double()
        gt = torch.ones((6, 3), device="cuda").double() if name == "top_log_probs" else None
        at = torch.where(y == -100, 0, y)
        index = torch.where(y[:, None] == -100, torch.arange(3, device="cuda"), got.top_indices._data)
        want, tol = _gradient(z, at, ones if name == "log_probs" else none, ones if name == "entropy" else none, gt,
                              index)
        live = (y != -100)
        assert ((x._grad.double() - want).abs() <= tol + U * want.abs())[live].all()
        assert (x._grad[2] == 0).all()


def test_gradients_match_differences():
    z, y = _logits(2, 37, torch.float32)
    w = torch.randn((2, 2), device="cuda").double()

    def loss(x):
        lp, _, entropy = _want(x, y)
        return (w[0] * lp.gather(-1, y[:, None])[:, 0] + w[1] * entropy).sum().item()

    x = _wrap(z, True)
    got = F.token_log_probs(x, _wrap(y))
    (got.log_probs * _wrap(w[0].float()) + got.entropy * _wrap(w[1].float())).sum().backward()
    for j in (0, 11, int(y[1])):
        step = torch.zeros((2, 37), device="cuda", dtype=torch.float64)
        step[1, j] = 1e-5
        slope = (loss(z.double() + step) - loss(z.double() - step)) / 2e-5
        # (the difference's own error: its third derivative, at most 6 (1 + ln V) |w|, times h^2 / 6, and 64 bits')
        assert abs(x._grad[1, j].item() - slope) < 1e-6 + 1e-5 * abs(slope)


def test_results_are_the_same_every_time_and_on_another_stream():
    z, y = _logits(5, 40003, torch.bfloat16)
    first = F.token_log_probs(_wrap(z), _wrap(y), 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side, side):
        with torch.cuda.stream(stream):
            again = F.token_log_probs(_wrap(z), _wrap(y), 20)
        stream.synchronize()
        for a, b in zip(first, again):
            assert torch.equal(a._data, b._data)


def test_a_captured_step_replays():
    z, y = _logits(4, 33000, torch.float16)
    up = torch.randn(4, device="cuda")

    def step(x):
        x.zero_grad()
        got = F.token_log_probs(x, _wrap(y), 5)
        (got.log_probs * _wrap(up) + got.entropy).sum().backward()
        return [got.log_probs._data, got.entropy._data, got.top_indices._data, x._grad]

    x = _wrap(z, True)
    held = F.token_log_probs(x, _wrap(y), 5)  # an eager graph of the same leaf, alive during the capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x)
    for seed in range(3):
        new, _ = _logits(4, 33000, torch.float16, seed=seed + 5)
        z.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        for a, b in zip(replayed, step(_wrap(new, True))):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    held.log_probs.sum().backward()


def test_a_model_scores_its_tokens():
    ts.seed(3)
    model = nn.TransformerLM(nn.TransformerConfig(61, dim=32, num_heads=2, num_layers=1, max_seq_len=16), device="hip")
    tokens = torch.randint(0, 61, (2, 7), device="cuda")
    targets = torch.randint(0, 61, (2, 7), device="cuda")
    targets[1, 4:] = -100
    got = model.token_log_probs(_wrap(tokens), _wrap(targets), 3)
    assert got.log_probs.shape == (2, 7) and got.top_indices.shape == (2, 7, 3)
    with ts.no_grad():
        _check(model(_wrap(tokens))._data[0], targets[0], 0, nn.functional.TokenLogProbs(
            _wrap(got.log_probs._data[0]), _wrap(got.entropy._data[0]), None, None))
    loss = model.loss(_wrap(tokens), _wrap(targets))
    assert abs(-got.log_probs._data.sum().item() / 11 - loss.item()) < 1e-5 * abs(loss.item()) + 1e-6
    (got.log_probs.sum() * -(1 / 11)).backward()
    grads = {n: p._grad.clone() for n, p in model.named_parameters()}
    for _, p in model.named_parameters():
        p.zero_grad()
    loss.backward()
    for n, p in model.named_parameters():
        scale = p._grad.double().norm()
        assert (grads[n].double() - p._grad.double()).norm() <= 1e-4 * scale, n


@pytest.mark.parametrize("rows,v", [(4097, 3999), (4096, 4097), (1, 4097), (2, 300007)])
def test_rows_a_wave_each_and_rows_of_many_parts(rows, v):
    z, y = _logits(rows, v, torch.bfloat16)
    for top in (0, 7, 64):
        print("token probs", rows, v, top, flush=True)
        _check(z, y, top, F.token_log_probs(_wrap(z), _wrap(y), top))
    up = torch.randn(rows, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    leaf = _wrap(z, True)
    F.token_log_probs(leaf, _wrap(y)).log_probs.backward(_wrap(up))
    want, tol = _gradient(z, y, up.double(), torch.zeros_like(up).double(), None, None)
    # (and dz rounds once, by 2^-8 at most)
    assert ((leaf.grad._data.double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-38).all()


def test_offsets_past_32_bits():
    rows, v = 43000, 50021  # 2.15e9 logits
    z = torch.zeros((rows, v), dtype=torch.bfloat16, device="cuda")
    z[-3:], y = _logits(3, v, torch.bfloat16)[0], torch.full((rows,), -100, device="cuda")
    y[-3:] = torch.tensor([5, 50020, 777], device="cuda")
    leaf = _wrap(z, True)
    got = F.token_log_probs(leaf, _wrap(y), 3)
    tail = F.TokenLogProbs(*(_wrap(x._data[-3:]) for x in got))
    _check(z[-3:], y[-3:], 3, tail)
    up = torch.zeros(rows, device="cuda")
    up[-3:] = torch.tensor([1.0, -2.0, 0.5], device="cuda")
    got.log_probs.backward(_wrap(up))
    want, tol = _gradient(z[-3:], y[-3:], up[-3:].double(), torch.zeros(3, device="cuda").double(), None, None)
    grad = leaf.grad._data
    assert ((grad[-3:].double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-38).all()
    assert not grad[:5].any() and not grad[rows // 2:rows // 2 + 5].any()


def _lowest(dtype):
    return torch.finfo(dtype).min


def _far_rows(v, dtype, low):
    """Rows of ordinary logits with `low` in front, in the middle, behind, everywhere but in one place and everywhere."""
    z, _ = _logits(6, v, dtype)
    z[0, :v // 2] = low
    z[1, v // 3:v // 3 + v // 5] = low
    z[2, v - v // 4:] = low
    z[3], z[3, (2 * v) // 3] = low, 1.0
    z[4] = low
    z[5, :min(v, 70)] = low
    # tokens with and without an ordinary logit
    return z, torch.tensor([0, v // 3, v - 1, (2 * v) // 3, v // 2, v - 1], device="cuda")


@pytest.mark.parametrize("dtype,low", [(d, low) for d in (torch.float32, torch.bfloat16)
                                       for low in (-1e7, -1e9, -1e10, -1e20, -1e30, _lowest(d))]
                         + [(torch.float16, _lowest(torch.float16))])
@pytest.mark.parametrize("v", [50, 2500, 30000])
def test_finite_masks_of_any_size(v, dtype, low):
    z, y = _far_rows(v, dtype, low)
    for top in (0, 5, 50):
        print("token probs", v, dtype, low, top, flush=True)
        _check(z, y, top, F.token_log_probs(_wrap(z), _wrap(y), top))
    g, gh = (torch.randn(6, generator=torch.Generator(device="cuda").manual_seed(v + n), device="cuda") for n in (1, 2))
    x = _wrap(z, True)
    got = F.token_log_probs(x, _wrap(y))
    (got.log_probs * _wrap(g) + got.entropy * _wrap(gh)).sum().backward()
    want, tol = _gradient(z, y, g.double(), gh.double(), None, None)
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + torch.finfo(dtype).smallest_normal
    assert ((x._grad.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("high", [1e7, 1e10, 1e30, 3e38])
@pytest.mark.parametrize("v", [50, 2500, 30000])
def test_large_logits(v, high, dtype):
    z, _ = _logits(5, v, dtype)
    z[0, v // 2] = high
    z[1, v - 1] = z[1, 0] = high
    z[2] = high
    z[3] = -high
    z[4] = torch.linspace(0, high, v, device="cuda").to(dtype)
    y = torch.tensor([v // 2, 1, 7, v - 1, v - 1], device="cuda")
    for top in (0, 5):
        print("token probs", v, dtype, high, top, flush=True)
        _check(z, y, top, F.token_log_probs(_wrap(z), _wrap(y), top))
    up = torch.tensor([1.0, -2.0, 0.5, 3.0, -1.0], device="cuda")
    x = _wrap(z, True)
    F.token_log_probs(x, _wrap(y)).log_probs.backward(_wrap(up))
    want, tol = _gradient(z, y, up.double(), torch.zeros(5, device="cuda").double(), None, None)
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + torch.finfo(dtype).smallest_normal
    assert ((x._grad.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("v", [50, 2500, 30000])
def test_large_upstream_gradients(v):
    z, y = _logits(3, v, torch.float32)
    z[:, v // 2] = -math.inf
    y = torch.where(y == v // 2, 0, y)
    g, gh = torch.tensor([1e12, -3e15, 0.0], device="cuda"), torch.tensor([-1e10, 1e20, 3e30], device="cuda")
    print("token probs vjp", v, flush=True)
    x = _wrap(z, True)
    got = F.token_log_probs(x, _wrap(y))
    (got.log_probs * _wrap(g) + got.entropy * _wrap(gh)).sum().backward()
    want, tol = _gradient(z, y, g.double(), gh.double(), None, None)
    assert ((x._grad.double() - want).abs() <= tol + U * (want.abs() + tol)).all()
    assert (x._grad[:, v // 2] == 0).all()


@pytest.mark.parametrize("rows,v", [((1 << 26) + 5, 3), ((1 << 24) + 3, 4097)])
def test_more_rows_than_a_grid_holds(rows, v):
    """Of a wave and of a workgroup a row: every row's results, and the gradient of the shorter ones."""
    z = torch.randn((rows, v) if v < 9 else (1, v), device="cuda", dtype=torch.float16).expand(rows, v)  # (long: one row)
    y = torch.arange(rows, device="cuda", dtype=torch.int32) % v
    y[5] = y[-2] = -100
    print("token probs", rows, v, flush=True)
    live = y >= 0
    with ts.no_grad():
        got = F.token_log_probs(_wrap(z), _wrap(y), 1)
    assert (got.log_probs._data[~live] == 0).all() and (got.top_indices._data[~live] == -1).all()
    d = _spread(v)
    if v > 9:
        lp, _, entropy = _want(z[:1], y[:1])
        want = lp[0].float()[y.long().clamp(min=0)]
        assert ((got.log_probs._data - want).abs() <= d + 5 * U * want.abs())[live].all()
        assert ((got.entropy._data - entropy.float()).abs() <= d + 2 * d * math.log(v) + 6 * U * math.log(v))[live].all()
        assert (got.top_indices._data[live] == z[0].argmax()).all()
        return
    for part in range(0, rows, 1 << 24):
        zz, at = z[part:part + (1 << 24)], y[part:part + (1 << 24)].long().clamp(min=0)
        want = torch.log_softmax(zz.double(), -1).gather(-1, at[:, None])[:, 0]
        close = (got.log_probs._data[part:part + (1 << 24)] - want).abs() <= d + 3 * U * want.abs().clamp(min=1)
        assert close[live[part:part + (1 << 24)]].all()
    leaf = _wrap(z, True)
    F.token_log_probs(leaf, _wrap(y)).log_probs.backward(_wrap(torch.ones(rows, device="cuda")))
    for part in range(0, rows, 1 << 24):
        zz, at = z[part:part + (1 << 24)], y[part:part + (1 << 24)].long()
        p = torch.softmax(zz.double(), -1)
        want = (torch.nn.functional.one_hot(at.clamp(min=0), v) - p) * (at >= 0)[:, None]
        tol = d + 30 * U + 2.0 ** -11 * want.abs() + 2.0 ** -25  # (f16: half a step, below its normal numbers 2^-25)
        assert ((leaf._grad[part:part + (1 << 24)].double() - want).abs() <= tol).all()
