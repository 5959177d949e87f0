"""Shapes over which the paged attention is run in each of the ways that it has.

A key is (dtype, channels, whether a column is a row, column blocks and waves of a workgroup,
whether there is more than one split); its shape (sequences, KV heads, query heads for each,
queries, positions, whether the sequences' lengths are spread up to that or all alike).  Keys
are every one that a search of some millions of shapes met; shapes are small ones of theirs.
"""

import ctypes

from tensorsmith_hip import _lib

SHAPES = {
    ("BF16", 32, False, 1, 4, False): (1, 1, 1, 2, 46, False),
    ("BF16", 32, False, 1, 4, True): (24, 1, 1, 2, 5931, False),
    ("BF16", 32, False, 1, 8, False): (1, 1, 1, 2, 201, False),
    ("BF16", 32, False, 1, 8, True): (1, 1, 2, 2, 2569, False),
    ("BF16", 32, False, 2, 4, False): (11, 4, 7, 40, 47, False),
    ("BF16", 32, False, 2, 4, True): (11, 3, 1, 18, 5178, False),
    ("BF16", 32, False, 2, 8, False): (10, 1, 4, 414, 1163, False),
    ("BF16", 32, False, 2, 8, True): (2, 12, 4, 13, 9316, False),
    ("BF16", 64, False, 1, 4, False): (1, 1, 2, 2, 45, False),
    ("BF16", 64, False, 1, 4, True): (1, 1, 1, 2, 1656, False),
    ("BF16", 64, False, 1, 8, False): (1, 1, 1, 2, 172, False),
    ("BF16", 64, False, 1, 8, True): (1, 1, 8, 2, 2177, False),
    ("BF16", 64, False, 2, 4, False): (41, 1, 7, 22, 45, False),
    ("BF16", 64, False, 2, 4, True): (2, 1, 2, 98, 2037, False),
    ("BF16", 64, False, 2, 8, False): (97, 4, 1, 17, 1175, True),
    ("BF16", 64, False, 2, 8, True): (1, 2, 7, 31, 10248, False),
    ("BF16", 64, True, 1, 4, False): (22, 3, 7, 17, 45, False),
    ("BF16", 64, True, 1, 4, True): (1, 2, 2, 190, 4483, False),
    ("BF16", 128, False, 1, 4, False): (1, 1, 1, 2, 56, False),
    ("BF16", 128, False, 1, 4, True): (1, 1, 1, 2, 1069, False),
    ("BF16", 128, False, 1, 8, False): (1, 1, 1, 2, 156, False),
    ("BF16", 128, False, 1, 8, True): (1, 1, 1, 2, 6849, False),
    ("BF16", 128, False, 2, 4, False): (14, 1, 7, 33, 46, False),
    ("BF16", 128, False, 2, 4, True): (1, 1, 3, 81, 1569, False),
    ("BF16", 128, False, 2, 8, False): (2, 4, 7, 34, 263, False),
    ("BF16", 128, False, 2, 8, True): (1, 2, 7, 19, 2378, False),
    ("BF16", 128, True, 1, 4, False): (11, 4, 2, 45, 46, False),
    ("BF16", 128, True, 1, 4, True): (1, 3, 3, 41, 1921, False),
    ("BF16", 256, False, 1, 4, False): (1, 1, 1, 2, 46, False),
    ("BF16", 256, False, 1, 4, True): (1, 1, 1, 3, 718, False),
    ("BF16", 256, False, 1, 8, False): (1, 1, 1, 2, 173, False),
    ("BF16", 256, False, 1, 8, True): (1, 1, 1, 2, 8696, False),
    ("BF16", 256, True, 1, 4, False): (1, 12, 3, 46, 48, False),
    ("BF16", 256, True, 1, 4, True): (1, 1, 7, 20, 1976, False),
    ("F16", 32, False, 1, 4, False): (1, 1, 1, 2, 50, False),
    ("F16", 32, False, 1, 4, True): (1, 1, 7, 2, 1983, False),
    ("F16", 32, False, 1, 8, False): (1, 1, 1, 2, 184, False),
    ("F16", 32, False, 1, 8, True): (1, 1, 2, 2, 2209, False),
    ("F16", 32, False, 2, 4, False): (25, 8, 4, 13, 46, False),
    ("F16", 32, False, 2, 4, True): (11, 3, 7, 3, 5345, False),
    ("F16", 32, False, 2, 8, False): (3, 4, 8, 172, 990, False),
    ("F16", 32, False, 2, 8, True): (24, 2, 7, 3, 9256, False),
    ("F16", 64, False, 1, 4, False): (1, 1, 1, 2, 46, False),
    ("F16", 64, False, 1, 4, True): (1, 1, 1, 2, 1388, False),
    ("F16", 64, False, 1, 8, False): (1, 1, 1, 2, 167, False),
    ("F16", 64, False, 1, 8, True): (1, 1, 1, 2, 6206, False),
    ("F16", 64, False, 2, 4, False): (2, 12, 7, 37, 46, False),
    ("F16", 64, False, 2, 4, True): (1, 1, 3, 130, 1957, False),
    ("F16", 64, False, 2, 8, False): (129, 2, 7, 5, 1561, True),
    ("F16", 64, True, 1, 4, False): (26, 4, 3, 22, 48, False),
    ("F16", 64, True, 1, 4, True): (49, 1, 3, 3, 2695, False),
    ("F16", 128, False, 1, 4, False): (1, 1, 1, 2, 48, False),
    ("F16", 128, False, 1, 4, True): (1, 1, 1, 2, 976, False),
    ("F16", 128, False, 1, 8, False): (1, 1, 1, 2, 149, False),
    ("F16", 128, False, 1, 8, True): (1, 1, 1, 2, 6668, False),
    ("F16", 128, False, 2, 4, False): (2, 12, 3, 43, 45, False),
    ("F16", 128, False, 2, 4, True): (1, 1, 4, 70, 1339, False),
    ("F16", 128, False, 2, 8, False): (194, 4, 2, 3, 291, True),
    ("F16", 128, True, 1, 4, False): (19, 3, 3, 23, 46, False),
    ("F16", 128, True, 1, 4, True): (1, 2, 1, 169, 1530, False),
    ("F16", 256, False, 1, 4, False): (1, 1, 1, 2, 47, False),
    ("F16", 256, False, 1, 4, True): (1, 1, 1, 2, 395, False),
    ("F16", 256, True, 1, 4, False): (1, 12, 7, 21, 45, False),
    ("F16", 256, True, 1, 4, True): (1, 2, 1, 165, 559, False),
    ("F32", 32, False, 1, 4, False): (1, 1, 1, 2, 47, False),
    ("F32", 32, False, 1, 4, True): (1, 1, 1, 2, 1615, False),
    ("F32", 32, False, 1, 8, False): (1, 1, 1, 2, 188, False),
    ("F32", 32, False, 1, 8, True): (1, 1, 3, 4, 2320, False),
    ("F32", 64, False, 1, 4, False): (1, 1, 1, 2, 50, False),
    ("F32", 64, False, 1, 4, True): (1, 1, 1, 3, 1205, False),
    ("F32", 64, False, 1, 8, False): (1, 1, 2, 2, 167, False),
    ("F32", 64, False, 1, 8, True): (1, 1, 1, 4, 6443, False),
    ("F32", 64, True, 1, 4, False): (19, 3, 7, 15, 45, False),
    ("F32", 64, True, 1, 4, True): (28, 1, 3, 3, 1674, False),
    ("F32", 128, False, 1, 4, False): (1, 1, 1, 3, 45, False),
    ("F32", 128, False, 1, 4, True): (1, 1, 1, 2, 757, False),
    ("F32", 128, False, 1, 8, False): (1, 1, 1, 2, 144, False),
    ("F32", 128, False, 1, 8, True): (1, 1, 1, 2, 8430, False),
    ("F32", 128, True, 1, 4, False): (31, 1, 7, 14, 47, False),
    ("F32", 128, True, 1, 4, True): (2, 1, 2, 77, 1171, False),
    ("F32", 256, False, 1, 4, False): (1, 1, 2, 2, 52, False),
    ("F32", 256, False, 1, 4, True): (1, 1, 1, 3, 279, False),
    ("F32", 256, True, 1, 4, False): (12, 1, 7, 14, 45, False),
    ("F32", 256, True, 1, 4, True): (1, 1, 3, 101, 400, False),
}


def lengths(shape):
    n, _, _, steps, keys, spread = shape
    return [max(steps, keys * (i + 1) // n) if spread else keys for i in range(n)]


def plan(dtype, d, shape, lens=None):
    """How the library runs it: ``_lib.Pages4Plan``."""
    n, heads, rep, steps, _, _ = shape
    lens = lengths(shape) if lens is None else lens
    out = _lib.Pages4Plan()
    desc = _lib.Pages4(0x10000, 1 << 20, heads, 64, d, 0x20000, n, 1 << 21)
    _lib.check(_lib.load().tsattn_pages4_attend_plan(desc, getattr(_lib, dtype), n, heads * rep, steps,
                                                     (ctypes.c_int32 * n)(*lens), out), "plan")
    return out


def key(dtype, d, p):
    return dtype, d, bool(p.wide), p.columns, p.waves, p.splits > 1
