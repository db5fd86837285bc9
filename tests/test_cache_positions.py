"""The positions that hk_cache_append takes without a rewind, by the rule its description states, on the ring of recent rows as
hk_cache lays it out (no GPU needed)."""
import random

import pytest

from paths import package


@pytest.mark.parametrize("seed", range(200))
def test_the_rule_names_positions_whose_rows_are_held(seed):
    """position p's row lies at p % 128 until position p + 128 takes the place: every earlier row of a block that the rule
    lets a call into is there, and a rewind is asked for only in a block that has been complete"""
    block, recent = package().CACHE_BLOCK, package().CACHE_RECENT
    r, ring = random.Random(seed), {}
    earliest = furthest = end = whole = 0
    for _ in range(30):
        pos = max(0, end - r.choice([0, r.randrange(recent), r.randrange(end + 1)]))
        count, first = r.choice([1, 2, 30, 100, 200]), pos - pos % block
        if max(earliest, furthest - recent) <= first and pos <= furthest:
            assert all(ring.get(p % recent) == p for p in range(first, pos))
        else:
            assert pos == first or first + block <= whole
            for p in range(first, pos):  # the rewind
                ring[p % recent] = p
            earliest, furthest = first, pos
        # (a call longer than the ring finds the first block's earlier rows apart from it)
        for p in range(pos, pos + count):
            ring[p % recent] = p
        end = pos + count
        furthest, whole = max(furthest, end), max(whole, end // block * block)
