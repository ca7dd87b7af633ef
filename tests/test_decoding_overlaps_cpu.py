"""Which states reorder_states takes for apart: against the bytes themselves."""
import random

import pytest
import torch

from pam_b200 import decoding


def _bytes(offset, groups, rows, by_group, by_row, size):
    return [(offset + g * by_group + r * by_row, offset + g * by_group + r * by_row + size) for g in range(groups) for r in range(rows)]


def _meet(a, b):
    return any(x < v and u < y for x, y in a for u, v in b)


def _refused(offsets, sizes, groups, rows, by_group, by_row):
    buffer = torch.zeros(4096, dtype=torch.uint8)
    states = [buffer[at:].as_strided((groups, rows, n), (by_group, by_row, 1)) for at, n in zip(offsets, sizes)]
    try:
        decoding._refuse_overlaps(states, list(sizes), torch.zeros(groups, rows, dtype=torch.int64))
    except ValueError:
        return True
    return False


def test_groups_that_end_between_rows():
    """The last row of a group of one state is the first of the next group of the other."""
    assert _refused((0, 4), (4, 4), 2, 2, 12, 8)
    assert not _refused((0, 4), (4, 4), 2, 2, 16, 8)
    assert not _refused((0, 4), (4, 4), 1, 2, 12, 8)


@pytest.mark.parametrize("seed", range(5))
def test_against_the_bytes(seed):
    rng, refused = random.Random(seed), 0
    for _ in range(400):
        groups, rows, size, other = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 6), rng.randint(1, 6)
        by_row = rng.randint(size, 24)
        by_group = rng.randint((rows - 1) * by_row + size, 4 * by_row + 20)
        if rng.random() < 0.3:                             # rows outside, groups within
            by_group = rng.randint(size, 24)
            by_row = rng.randint((groups - 1) * by_group + size, 4 * by_group + 20)
        apart = rng.randint(0, 60)
        mine = [_bytes(0, groups, rows, by_group, by_row, size), _bytes(apart, groups, rows, by_group, by_row, other)]
        # (each state's own rows are checked for themselves: the second one's may meet where it is wider)
        alone = any(_meet(s[i:i + 1], s[i + 1:]) for s in mine for i in range(len(s)))
        meet = _meet(*mine)
        got = _refused((0, apart), (size, other), groups, rows, by_group, by_row)
        refused += meet and not alone
        assert got if meet or alone else not got
    assert refused > 20
