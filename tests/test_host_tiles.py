"""Plans of tiles and what a launch of them refuses (csrc/tile.hpp), against a stand-in of the HIP
runtime: no GPU is used."""
import ctypes
import itertools
import os

import hostrun

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "build", "libtiletest.so")


def _launches(cases):
    lib = ctypes.CDLL(LIB)
    lib.tile_error.restype = ctypes.c_char_p
    out = []
    for c in cases:
        hostrun.clear_launches()
        rc = lib.tile_launch(*c)
        out.append((rc, lib.tile_error().decode() if rc else "", sum(hostrun.launches().values())))
    return out


def test_a_split_without_a_stage_is_not_launched():
    """it would have no last stage to repeat: its loads would begin before the operands"""
    cases = [(3, 4, 2, 1), (3, 4, 4, 3), (1, 1, 16, 15), (3, 4, 0, 3), (1, 1, 1, 0)]
    for c, (rc, text, n) in zip(cases, hostrun.call(_launches, cases)):
        assert rc < 0 and "without a stage" in text and n == 0, (c, rc, text, n)
    for rc, _, n in hostrun.call(_launches, [(3, 4, 1, 1), (3, 4, 2, 2), (1, 1, 16, 16), (1, 1, 16, 1000)]):
        assert rc == 0 and n == 1


def test_more_tiles_than_a_launch_takes():
    (rc, text, n), = hostrun.call(_launches, [(1 << 16, 1 << 16, 1, 5)])
    assert rc < 0 and "more tiles" in text and n == 0


KINDS = [[(64, 32, 256), (64, 64, 128), (128, 128, 128), (256, 256, 128)], [(64, 32, 128), (64, 64, 128), (128, 128, 128)]]
TIMES = [0.56, 0.38, 0.36, 0.23, 0.57, 0.62, 0.9, 1.5]


def _plans(sizes):
    lib = ctypes.CDLL(LIB)
    out = []
    for kinds in KINDS:
        flat = (ctypes.c_uint32 * (3 * len(kinds)))(*itertools.chain(*kinds))
        times = (ctypes.c_float * (2 * len(kinds)))(*TIMES[:2 * len(kinds)])
        for cols, rows, halves, row_bytes in sizes:
            plan = (ctypes.c_uint32 * 5)()
            lib.tile_plan(flat, times, len(kinds), ctypes.c_uint64(cols), ctypes.c_uint64(rows), halves, ctypes.c_uint64(row_bytes),
                          ctypes.c_uint64(cols * rows * (1 + halves)), plan)
            out.append((kinds, (cols, rows, halves, row_bytes), list(plan)))
    return out


def test_plans_cover_their_products():
    """whole tiles for every row and column, stages for the whole reduction, two or more in each split"""
    lengths = [1, 2, 31, 64, 65, 300, 1000, 4096, 16384, 1 << 20]
    reductions = [2, 10, 128, 254, 256, 258, 500, 512, 514, 1024, 2046, 4098, 8192, 131072, 1 << 21]
    sizes = [(c, r, h, b) for c in lengths for r in lengths for h in (0, 1) for b in reductions]
    split = 0
    for kinds, (cols, rows, halves, row_bytes), (kind, ta, tb, splits, steps) in hostrun.call(_plans, sizes):
        na, nb, kb = kinds[kind]
        assert (ta - 1) * na < cols <= ta * na and (tb // (1 + halves) - 1) * nb < rows <= tb // (1 + halves) * nb
        assert (steps - 1) * kb < row_bytes <= steps * kb
        assert splits == 1 or steps // splits >= 2, (cols, rows, row_bytes, splits, steps)
        split += splits > 1
    assert split > 100
