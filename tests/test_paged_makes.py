"""The ways in which the paged attention is run, as its plan tells them: every kernel that
can be launched has a shape, which the GPU tests take against float64."""

from __future__ import annotations

import ctypes
import random

import pytest

pytest.importorskip("torch")

from paged_makes import SHAPES, key, lengths, plan  # noqa: E402
from tensorsmith_hip import _lib  # noqa: E402


@pytest.mark.parametrize("make", SHAPES, ids=lambda x: "-".join(map(str, x)))
def test_a_shape_is_run_as_its_key_says(make):
    dtype, d, *_ = make
    p = plan(dtype, d, SHAPES[make])
    assert key(dtype, d, p) == make
    assert p.split % 32 == 0 and 0 < p.split <= 4096
    assert p.splits == -(-max(lengths(SHAPES[make])) // p.split)


def test_the_shapes_cover_every_kernel():
    """Columns of groups: one block or two with four waves or eight, but no two blocks of fp32 or of 256
    channels, and no eight waves of 256 channels but in bf16; columns of rows from 64 channels on.  Each
    with one split and with several, but for a few that no shape was found for."""
    kernels = set()
    for dtype in ("F32", "F16", "BF16"):
        for d in (32, 64, 128, 256):
            kernels |= {(dtype, d, False, c, w) for c in (1, 2) for w in (4, 8)
                        if not (c == 2 and (dtype == "F32" or d == 256)) and not (w == 8 and d == 256 and dtype != "BF16")}
            if d > 32:
                kernels.add((dtype, d, True, 1, 4))
    assert {make[:5] for make in SHAPES} == kernels
    every = {k + (s,) for k in kernels for s in (False, True)}
    assert every - set(SHAPES) == {("F16", 64, False, 2, 8, True), ("F16", 128, False, 2, 8, True)}


def test_any_shapes_way_is_among_them():
    rng = random.Random(7)
    for _ in range(4000):
        dtype, d = rng.choice(("F32", "F16", "BF16")), rng.choice((32, 64, 128, 256))
        n, keys = int(2 ** rng.uniform(0, 7)), int(2 ** rng.uniform(0, 15))
        shape = (n, rng.choice((1, 2, 4, 8, 12)), rng.choice((1, 2, 4, 7, 8)), int(2 ** rng.uniform(0, 10)), keys, False)
        lens = [rng.randint(0, keys) for _ in range(n)] if rng.random() < 0.5 else None
        assert key(dtype, d, plan(dtype, d, shape, lens)) in SHAPES, (dtype, d, shape, lens)


def test_sizes_without_a_plan_are_refused():
    lib, out, lens = _lib.load(), _lib.Pages4Plan(), (ctypes.c_int32 * 2)(5, 6)
    desc = lambda **kw: _lib.Pages4(0x10000, 8, kw.get("heads", 2), 64, kw.get("dim", 64), 0x20000, 2, 4)  # noqa: E731
    call = lambda d=desc(), dtype=_lib.F16, n=2, heads=4, steps=1, lens=lens, out=out: (  # noqa: E731
        lib.tsattn_pages4_attend_plan(d, dtype, n, heads, steps, lens, out))
    assert call() == 0 and (out.sequences, out.rows, out.splits) == (2, 2, 1)
    for bad in (call(None), call(desc(dim=48)), call(dtype=_lib.F64), call(n=0), call(heads=3), call(heads=0),
                call(steps=0), call(steps=1 << 20), call(lens=None), call(lens=(ctypes.c_int32 * 2)(-1, 5)),
                call(lens=(ctypes.c_int32 * 2)(1 << 28, 5)), call(out=None)):
        assert bad == _lib.ERR_INVALID and "no plan" in _lib.last_error()
