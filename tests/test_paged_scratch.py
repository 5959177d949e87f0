"""The paged attention's scratch: bounded whatever the sequences' lengths, and as it was
where it fits."""

from __future__ import annotations

import ctypes
import importlib

import numpy as np
import pytest

pytest.importorskip("torch")

from tensorsmith_hip import _lib  # noqa: E402

P = importlib.import_module("tensorsmith_hip.nn.paged")
F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16


def scratch(dtype, hkv, dim, heads, steps, lens):
    desc = _lib.Pages4(0x10000, 1 << 20, hkv, 64, dim, 0x20000, len(lens), 1 << 21)
    return _lib.load().tsattn_pages4_attend_workspace(desc, dtype, len(lens), heads, steps,
                                                      (ctypes.c_int32 * len(lens))(*lens))


@pytest.mark.parametrize("dtype,hkv,dim,heads,steps,lens", [
    (F32, 8, 128, 8, 1024, (131072,) + (2000,) * 63),
    (BF16, 8, 256, 8, 1024, (131072,) + (2000,) * 63),
    (BF16, 8, 128, 32, 32, (1 << 20,) + (512,) * 255),
    (F16, 8, 128, 32, 8, (512,) * 300 + (1 << 22,) + (512,) * 300),
    (BF16, 8, 256, 256, 8192, (131072,)),
    (F16, 12, 256, 96, 1000, (100, 1 << 20, 0, 300_000)),
    (F32, 4096, 256, 4096, 1, (1 << 14,) * 3),
    (F32, 1, 32, 8, 1 << 15, (1 << 27,)),
])
def test_it_is_at_most_four_gigabytes(dtype, hkv, dim, heads, steps, lens):
    need = scratch(dtype, hkv, dim, heads, steps, lens)
    assert 0 < need <= 1 << 32
    # a part holds a sequence's rows, or 32 of them, at least
    assert need >= 4 * min(heads // hkv * steps, 32) * hkv * -(-max(lens) // 4096) * (dim + 2)


def test_one_sequence_of_few_rows_takes_what_it_needs():
    """As many splits as the longest sequence has for every sequence of the launch."""
    for n in (1, 3, 256):
        need = scratch(BF16, 8, 128, 32, 1, (131072,) + (1000,) * (n - 1))
        splits = need // (4 * n * 8 * 4 * 130)
        assert need == 4 * n * 8 * 4 * 130 * splits and splits >= 32


def test_the_rule_counts_positions_that_are_there():
    """A long sequence beside short ones reads its codes: their partial sums are few, whatever a launch
    would lay out for all of them; the sums of one over the limit are not."""
    lens = np.array((131072,) + (2000,) * 63, np.int32)
    assert P._reads_codes(1024, 8, 128, True, lens)
    assert scratch(F32, 8, 128, 8, 1024, lens.tolist()) <= 1 << 32
    assert not P._reads_codes(1 << 16, 8, 128, True, lens)
