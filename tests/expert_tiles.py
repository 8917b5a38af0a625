"""Which tiles the experts' products run for given counts: the plan is the library's own choice (asked for on the host), the
walk of the blocks over their lists is stated again here."""
import ctypes
from collections import Counter
from typing import NamedTuple

from mooncake_amd import _lib

XCDS = 8
STEP = 128          # bytes of a row per K step


class Shape(NamedTuple):
    weight_rows: int        # 256 or 128
    blocks: int             # of 32 rows
    streamed: bool = False


class Tiles(NamedTuple):
    plan: tuple             # rows of a tile at most, weight rows
    runs: Counter           # tiles of each shape
    behind: Counter         # of those: whose first loads were issued by a tile of the same shape in front of it
    switches: int           # times that a block goes on with another shape


def plan(counts, rows_per_expert, columns, row_bytes, fp8, gate_up, grid):
    out = [ctypes.c_int32() for _ in range(4)]
    _lib.check(_lib.lib().mc_ep_debug_expert_plan((ctypes.c_int32 * max(len(counts), 1))(*counts), len(counts), rows_per_expert, columns,
                                                  row_bytes, int(fp8), int(gate_up), grid, *(ctypes.byref(o) for o in out)))
    return tuple(o.value for o in out)


def stages(shape):
    return 4 if shape.weight_rows < 256 else 3 if shape.blocks <= 4 else 2


def walk(counts, rows_per_expert, columns, row_bytes, fp8, gate_up, cus=256):
    grid = cus // XCDS * XCDS
    most, weight_rows, row_tiles, streamed = plan(counts, rows_per_expert, columns, row_bytes, fp8, gate_up, grid)
    counts = [min(max(n, 0), rows_per_expert) for n in counts]
    tile_columns = weight_rows // 2 if gate_up else weight_rows
    across = -(-columns // tile_columns)
    steps = -(-row_bytes // STEP)
    tiles = []                                  # in the order of the list
    for n in counts:
        if not n:
            continue
        down = -(-n // most)
        each = -(-n // down)
        tiles += [Shape(weight_rows, -(-min(each, n - m * each) // 32), bool(streamed)) for _ in range(across) for m in range(down)]
    assert len(tiles) == row_tiles * across and all(s.blocks * 32 <= most for s in tiles)
    runs, behind, switches = Counter(tiles), Counter(), 0
    for block in range(grid):
        xcd = block % XCDS
        t, end = len(tiles) * xcd // XCDS + block // XCDS, len(tiles) * (xcd + 1) // XCDS
        mine = tiles[t:end:grid // XCDS]
        for a, b in zip(mine, mine[1:]):
            if a == b and steps >= stages(a):
                behind[b] += 1
            switches += a != b
    return Tiles((most, weight_rows), runs, behind, switches)


def products(counts, rows_per_expert, hidden, intermediate, fp8, cus=256):
    """(gate_up, down) of a call of expert_mlp."""
    size = 1 if fp8 else 2
    return (walk(counts, rows_per_expert, intermediate, hidden * size, fp8, True, cus),
            walk(counts, rows_per_expert, hidden, intermediate * size, fp8, False, cus))


def every_shape(fp8, gate_up):
    """All tile shapes that the kernel has."""
    wide = [Shape(256, b) for b in range(1, 9)] + [Shape(256, 1, True)]
    return set(wide + ([] if fp8 and gate_up else [Shape(128, b) for b in range(1, 5)]))


class Case(NamedTuple):
    """Experts of hidden x intermediate whose rows rise from `low` to `high` over the first 1 / `steep` of them: tiles of one
    shape follow each other, and every shape up to the largest comes."""
    fp8: bool
    experts: int
    hidden: int
    intermediate: int
    low: int
    high: int
    steep: int = 1

    @property
    def counts(self):
        return [min(self.high, self.low + e * self.steep * (self.high - self.low) // (self.experts - 1)) for e in range(self.experts)]

    @property
    def rows(self):
        return self.high + 3

    @property
    def name(self):
        return f"{'fp8' if self.fp8 else 'bf16'}-{self.experts}x{self.hidden}x{self.intermediate}-{self.low}to{self.high}"

    def products(self, cus=256):
        return products(self.counts, self.rows, self.hidden, self.intermediate, self.fp8, cus)


# Together every tile shape of both products and types, each with tiles whose loads began behind another's (test_expert_plan.py)
CASES = [Case(False, 48, 256, 1280, 1, 256), Case(False, 64, 1664, 256, 1, 224), Case(False, 40, 1920, 256, 220, 250),
         Case(False, 64, 1280, 640, 1, 20), Case(False, 137, 384, 3840, 1, 128), Case(False, 60, 5120, 640, 1, 126, 4),
         Case(True, 64, 512, 1024, 1, 250), Case(True, 64, 1920, 384, 1, 256), Case(True, 40, 1664, 1024, 1, 20),
         Case(True, 92, 640, 7424, 1, 110)]


def covered(cases, fp8, product, cus=256):
    """The tile shapes of a product (0 gate_up, 1 down) that the cases run behind another tile of the same shape."""
    return {shape for case in cases if case.fp8 == fp8 for shape in case.products(cus)[product].behind}
