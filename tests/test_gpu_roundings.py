"""Windowed and cached attention in 16 bits within their own roundings, element by element.

u is half a step of the type (2^-11 in f16, 2^-8 in bf16), e = 2^-24 fp32's; sizes are sums of
absolute values in float64, P the exact softmax, P V its output O.

Scores are sums of D products in fp32: off by at most D e of sum |q k|.  In log2 units a product
and an exponential follow, so that P is off by at most f = 2 (D + 4) e scale max sum |q k| + 2^-20
of itself (twice: its own exponential and the row's sum), sums of n terms by n e of their size.
* O: P rounds to the type once (u; over int8 codes and f16 queries to two bf16 parts, 2^-16; codes
  times bf16's P: u), the sum of P not at all, the result once: |dO| <= (u + f + n e) sum P |V| + u |O|.
* dV = P^T dO: the same with sum P |dO|.
* delta = dO O, O as it was before its own rounding (two parts of the type keep 2 u^2 of it), off by
  E = sum_c |dO_c| (u + f + n e + 2 u^2) (sum P |V|)_c; dP by D e of sum |dO V|.
* dS = P (dP - delta) rounds once: off by u |dS| + P E + P (f + 2 D e) (sum |dO V| + sum |dO O|);
  dK and dQ are those times scale |q| (|k|), and u of themselves.
What is below f16's normal numbers is off by 2^-25 instead: of P and dS a term each.  Each bound is
taken with a hundredth more for the products of these terms.
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

E = 2.0 ** -24


def _wrap(x, grad=False):
    return ts.Tensor(x, device="hip", requires_grad=grad)


def _draw(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _seen(sq, sk, window, sinks):
    i, j = torch.arange(sk - sq, sk, device="cuda")[:, None], torch.arange(sk, device="cuda")[None]
    return (j <= i) & ((j > i - window) | (j < sinks))


def _within(name, got, want, bound):
    off = (got.double() - want).abs()
    worst = (off / (1.01 * bound)).max().item()
    print(f"{name}: {worst:.2f} of its bound", flush=True)
    assert (off <= 1.01 * bound).all(), (name, worst)


def _forward(q, k, v, seen):
    """P, O, sum P |V|, f in float64 (k, v a head each)."""
    d, scale = q.shape[-1], 1 / math.sqrt(q.shape[-1])
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    f = 2 * (d + 4) * E * scale * torch.matmul(q.abs(), k.abs().transpose(-1, -2).contiguous()).max() + 2.0 ** -20
    p = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
    return p, torch.matmul(p, v), torch.matmul(p, v.abs()), f


def _units(dtype):
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks,d", [(4, 0, 64), (20, 3, 128), (90, 0, 32), (300, 40, 64)])
def test_windows_are_within_their_roundings(window, sinks, d, dtype):
    b, hq, hkv, s = 1, 4, 2, 500
    q, k, v, up = (_draw(b, h, s, d, dtype=dtype, seed=n) for n, h in enumerate((hq, hkv, hkv, hq)))
    leaves = [_wrap(x, True) for x in (q, k, v)]
    print("window", window, sinks, d, dtype, flush=True)
    out = nn.scaled_dot_product_attention(*leaves, is_causal=True, enable_gqa=True, window=window, sinks=sinks)
    out.backward(_wrap(up))
    u, tiny = _units(dtype)
    rep, scale = hq // hkv, 1 / math.sqrt(d)
    q, up = q.double(), up.double()
    k, v = (x.double().repeat_interleave(rep, 1) for x in (k, v))
    seen = _seen(s, s, window, sinks)
    p, o, size, f = _forward(q, k, v, seen)
    n = seen.sum(-1).max().item()
    _within("out", out._data, o, (u + f + n * E) * size + u * o.abs() + tiny * (n * v.abs().max() + 1))
    across = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    group = lambda x: x.reshape(b, hkv, rep, s, d).sum(2)  # noqa: E731
    rows = seen.sum(-2).max().item() * rep
    dv, dv_size = group(torch.matmul(across(p), up)), group(torch.matmul(across(p), up.abs()))
    _within("dv", leaves[2]._grad, dv,
            (u + f + rows * E) * dv_size + u * dv.abs() + tiny * (rows * up.abs().max() + 1))
    dp, dp_size = torch.matmul(up, across(v)), torch.matmul(up.abs(), across(v.abs()))
    delta = (up * o).sum(-1, keepdim=True)
    off = (up.abs() * size).sum(-1, keepdim=True) * (u + f + n * E + 2 * u * u)
    ds = p * (dp - delta)
    ds_off = u * ds.abs() + p * off + p * (f + 2 * d * E) * (dp_size + (up * o).abs().sum(-1, keepdim=True)) + tiny * seen
    for name, leaf, mine, other, terms in (("dq", leaves[0], lambda x: x, k, n),
                                           ("dk", leaves[1], across, q, rows)):
        fold = group if name == "dk" else lambda x: x
        want = fold(torch.matmul(mine(ds), other)) * scale
        bound = fold(torch.matmul(mine(ds_off + terms * E * ds.abs()), other.abs())) * scale
        _within(name, leaf._grad, want, bound + u * (want.abs() + bound) + tiny)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,rep,tokens,length", [(3, 4, 1, 700), (2, 1, 5, 90), (40, 4, 33, 600)])
def test_cached_attention_is_within_its_roundings(b, rep, tokens, length, d, int8, dtype):
    hkv, window, sinks = 4, 60, 4
    cache = nn.KVCache(b, hkv, d, length, device="hip", dtype=dtype, quantized=int8)
    q = _draw(b, hkv * rep, tokens, d, dtype=dtype, seed=3)
    with ts.no_grad():
        cache.append(*(_wrap(_draw(b, hkv, length, d, dtype=dtype, seed=n)) for n in (1, 2)))
        print("cached", b, rep, tokens, length, d, int8, dtype, flush=True)
        got = nn.cached_attention(_wrap(q), cache, window=window, sinks=sinks)._data
    keys, values, ks, vs = cache.storage
    k, v = ((x.double() if s is None else x.double() * s.double()).repeat_interleave(rep, 1)
            for x, s in ((keys, ks), (values, vs)))
    u, tiny = _units(dtype)
    _, o, size, f = _forward(q.double(), k, v, _seen(tokens, length, window, sinks))
    n = window + sinks
    # (scales multiply a score and P: 2 e more)
    inner, terms = (2.0 ** -16 + 2 * E, 0.0) if int8 and dtype == torch.float16 else (u + 2 * E, 0.0 if int8 else tiny)
    _within("out", got, o, (inner + f + n * E) * size + u * o.abs() + terms * n * v.abs().max() + tiny)
