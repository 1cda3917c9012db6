"""CPU: which kernel a dense product takes on the 148 SMs of a B200.  The tables name, for every tile that is compiled and every form it is compiled in, ragged
shapes that select it; tests/test_gpu_dense_tiles.py runs them.  A retuned constant that moves a shape to another tile shows here."""
import ctypes
import random

import pytest

SMS = 148
# (m, n, k): the tile {CTAs, columns, ways k is split}.  Persistent tiles with more tiles than CTAs (several turns), odd numbers of k blocks.
LINEAR = {(261, 8984, 112): (1, 128, 1), (100, 1856, 408): (1, 128, 2), (90, 960, 1472): (1, 128, 4), (929, 7080, 144): (2, 192, 1), (1500, 4104, 1544): (2, 192, 1),
          (2835, 7336, 104): (2, 256, 1), (2500, 5128, 1160): (2, 256, 1), (1702, 656, 6128): (2, 256, 2)}
LINEAR_ODD = {(309, 8485, 104): (1, 128, 1), (100, 1873, 432): (1, 128, 2), (90, 993, 1440): (1, 128, 4), (3283, 6593, 104): (2, 256, 1), (1702, 655, 6124): (2, 256, 2)}
# (m, inter, k)
GATED = {(200, 4000, 120): (1, 128, 1), (130, 1200, 1696): (1, 128, 2), (90, 464, 1656): (1, 128, 4), (7267, 480, 104): (2, 192, 1), (1500, 2056, 776): (2, 192, 1),
         (401, 7168, 648): (2, 256, 1), (136, 3272, 5600): (2, 256, 2)}
GATED_ODD = {(200, 4001, 128): (1, 128, 1), (130, 1201, 1720): (1, 128, 2), (90, 481, 1544): (1, 128, 4), (551, 6003, 656): (2, 256, 1), (136, 3269, 5600): (2, 256, 2)}
FP8 = {(277, 8296, 128): (1, 128, 1), (100, 1960, 512): (1, 128, 2), (90, 928, 1920): (1, 128, 4), (1665, 4016, 256): (2, 192, 1), (5127, 1296, 384): (2, 192, 1)}
# (m, n, k) of a projection: the tiles of dx [m, k] = dz w and of dw [n, k] = dz^T x
BACKWARD = {(265, 24, 7640): ((1, 128, 1), (1, 128, 1)), (21, 1768, 4768): ((1, 128, 2), (1, 128, 1)), (90, 1448, 1016): ((1, 128, 4), (1, 128, 1)),
            (1755, 24, 4784): ((1, 128, 1), (1, 128, 2)), (1411, 24, 936): ((1, 128, 1), (1, 128, 4)), (3501, 648, 1928): ((2, 256, 1), (1, 128, 1)),
            (137, 5304, 4840): ((2, 256, 2), (1, 128, 1)), (645, 7320, 928): ((1, 128, 2), (2, 256, 1)), (5393, 4752, 144): ((1, 128, 1), (2, 256, 2))}
BACKWARD_ODD = {(3501, 649, 1929): ((2, 256, 1), (1, 128, 1)), (137, 5303, 4839): ((2, 256, 2), (1, 128, 1)), (645, 7321, 929): ((1, 128, 2), (2, 256, 1)),
                (5393, 4751, 145): ((1, 128, 1), (2, 256, 2))}


def tile(lib, m, n, k, *, gated=0, a_mn=0, b_mn=0, fp8=0, residual=0, single=0, sms=SMS):
    t = (ctypes.c_int * 3)()
    assert lib.b200_dense_tile(m, n, k, gated, a_mn, b_mn, fp8, residual, single, sms, ctypes.addressof(t)) == 0
    return tuple(t)


def picks(lib, sms=SMS):
    """(what, expected tile, tile on this many SMs) of every shape in the tables."""
    out = []
    for table, odd in ((LINEAR, 0), (LINEAR_ODD, 1)):
        out += [(("linear", s), want, tile(lib, *s, single=odd, residual=1, sms=sms)) for s, want in table.items()]
    for table, odd in ((GATED, 0), (GATED_ODD, 1)):
        out += [(("gated", s), want, tile(lib, s[0], 2 * s[1], s[2], gated=1, single=odd, sms=sms)) for s, want in table.items()]
    out += [(("fp8", s), want, tile(lib, *s, fp8=1, residual=1, sms=sms)) for s, want in FP8.items()]
    for table, odd in ((BACKWARD, 0), (BACKWARD_ODD, 1)):
        for (m, n, k), (dx, dw) in table.items():
            out += [(("dx", (m, n, k)), dx, tile(lib, m, k, n, b_mn=1, single=odd, sms=sms)), (("dw", (m, n, k)), dw, tile(lib, n, k, m, a_mn=1, b_mn=1, single=odd, sms=sms))]
    return out


def test_tables(mods):
    wrong = [p for p in picks(mods.lib.lib()) if p[1] != p[2]]
    assert not wrong, wrong


def test_tables_reach_every_tile():
    every = {(1, 128, 1), (1, 128, 2), (1, 128, 4), (2, 256, 1), (2, 256, 2)}
    assert set(LINEAR.values()) == set(GATED.values()) == every | {(2, 192, 1)}
    assert set(LINEAR_ODD.values()) == set(GATED_ODD.values()) == every  # a row of single values takes no 192-wide tile
    assert set(FP8.values()) == {(1, 128, 1), (1, 128, 2), (1, 128, 4), (2, 192, 1)}
    assert {t for t, _ in BACKWARD.values()} == every and {t for _, t in BACKWARD.values()} == every


def test_every_compiled_choice_is_taken(mods):
    """What is compiled is reached, on SM counts beside this one too, and nothing else is chosen."""
    lib, rng, seen = mods.lib.lib(), random.Random(2), set()
    for _ in range(20000):
        m, n, k = (int(2 ** rng.uniform(4.2, hi)) for hi in (14, 13.5, 13))
        form = rng.choice(["plain", "odd", "gated", "fp8", "dx", "dw"])
        kw = {"plain": {}, "odd": {"single": 1}, "gated": {"gated": 1}, "fp8": {"fp8": 1}, "dx": {"b_mn": 1}, "dw": {"a_mn": 1, "b_mn": 1}}[form]
        t = tile(lib, m, n // 2 * 2 + 2, k // 128 * 128 + 128, residual=rng.randint(0, 1) if form in ("plain", "fp8") else 0, sms=rng.choice([SMS, SMS, 132, 160]), **kw)
        seen.add((form, t))
    five = {(1, 128, 1), (1, 128, 2), (1, 128, 4), (2, 256, 1), (2, 256, 2)}
    want = {(f, t) for f in ("plain", "gated", "odd", "dx", "dw") for t in five} | {(f, (2, 192, 1)) for f in ("plain", "gated", "fp8")}
    assert {s for s in seen if s[1] != (0, 0, 0)} == want | {("fp8", t) for t in five if t[1] == 128}


def test_few_rows_and_refusals(mods):
    lib = mods.lib.lib()
    assert tile(lib, 16, 512, 512) == tile(lib, 16, 512, 512, fp8=1) == tile(lib, 1, 512, 512, gated=1) == (0, 0, 0)
    assert tile(lib, 16, 512, 512, b_mn=1) != (0, 0, 0) and tile(lib, 17, 512, 512) != (0, 0, 0)
    t = (ctypes.c_int * 3)()
    assert lib.b200_dense_tile(0, 8, 8, 0, 0, 0, 0, 0, 0, SMS, ctypes.addressof(t)) == -1
    assert lib.b200_dense_tile(8, 8, 8, 0, 0, 0, 0, 0, 0, SMS, None) == -1
    assert lib.b200_dense_tile(8, (1 << 30) + 1, 8, 0, 0, 0, 0, 0, 0, SMS, ctypes.addressof(t)) == -6
