"""What the joining kernels of the cache attention read (host side of the same functions, no GPU): for a table that the main kernel has written, the slots that
its pieces went to; for one that it has left as the workspace came, nothing outside the workspace's slots."""
import random

import pytest

from delta_matching_b200 import _lib

INT = (-(1 << 31), (1 << 31) - 1)


def _slots(many_rows, x, y, grid):
    L = _lib.lib()
    n = L.dm_dbg_cache_join_slots(many_rows, x, y, grid, -1)
    return [L.dm_dbg_cache_join_slots(many_rows, x, y, grid, i) for i in range(n)]


@pytest.mark.parametrize("many_rows", [0, 1])
@pytest.mark.parametrize("grid", [1, 2, 148, 444])
def test_any_entry_stays_inside(many_rows, grid):
    rng = random.Random(grid)
    room = grid * (2 if many_rows else 8)
    edge = [*INT, -1, 0, 1, room - 1, room, room + 1, grid - 1, grid, 4 * grid, 0x7FC00000, 0x3F800000]
    pairs = [(x, y) for x in edge for y in edge] + [(rng.randint(*INT), rng.randint(*INT)) for _ in range(500)]
    pairs += [(rng.randrange(-2, room + 2), rng.randrange(-2, room + 2)) for _ in range(500)]
    for x, y in pairs:
        got = _slots(many_rows, x, y, grid)
        assert len(got) <= grid + 1 and all(0 <= s < room for s in got), (x, y, got)
        assert len(set(got)) == len(got) or x // 2 == (y if many_rows else y >> 1)


def test_pieces_of_ctas():
    """The first piece, then the first slot of every CTA up to the last."""
    assert _slots(1, 7, 6, 148) == [7, 8, 10, 12]
    assert _slots(1, 6, 4, 148) == [6, 8]
    assert _slots(1, -1, 4, 148) == []


def test_pieces_of_warps():
    """Warp w writes slots 2 w and 2 w + 1; a CTA's warps that end in one unit are joined in the first one's slot."""
    assert _slots(0, 2 * 5 + 1, 2 * 14, 148) == [11, 16, 24]             # warp 5's second piece (6, 7 joined to it); CTA 2 joined; CTA 3's warps 12 - 14 joined
    assert _slots(0, 2 * 5, 2 * 14 + 1, 148) == [10, 16, 24, 28]         # warp 14 went on with another unit: its own slot
    assert _slots(0, 2 * 5, 2 * 12 + 1, 148) == [10, 16, 24]             # it is the first of its CTA: nothing joined there
    assert _slots(0, 2 * 5, 2 * 7 + 1, 148) == [10, 14]
    assert _slots(0, 2 * 5, 2 * 8, 148) == [10, 16]


def test_refuses():
    L = _lib.lib()
    assert L.dm_dbg_cache_join_slots(0, 0, 0, 0, -1) == -1 and "grid" in _lib.last_error()
    assert L.dm_dbg_cache_join_slots(1, 0, 1, 148, 2) == -1 and "piece 2 of 2" in _lib.last_error()
