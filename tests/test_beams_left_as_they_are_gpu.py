"""Beams whose parent, page or row is not there stay as they are; all others move: every page, table entry and state record, to the bit."""
from __future__ import annotations

import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops.beams import beam_reorder

pytestmark = pytest.mark.gpu
PAGE, PAGES, ROWS = 8, 40, 12


def expected(parents, lengths, table, cache, state, rows):
    old_table, old_cache, old_state = table.clone(), cache.clone(), state.clone()
    groups, beams = parents.shape
    for g in range(groups):
        full, filled = divmod(max(0, int(lengths[g])), PAGE)
        for j in range(beams):
            p, i = int(parents[g, j]), g * beams + j
            source = g * beams + (p if 0 <= p < beams else j)
            table[i, :full] = old_table[source, :full]
            if filled and full < table.shape[1]:
                to, at = int(old_table[i, full]), int(old_table[source, full])
                if 0 <= to < PAGES and 0 <= at < PAGES:
                    cache[:, to, :, :filled] = old_cache[:, at, :, :filled]
            to, at = int(rows[i]), int(rows[source])
            if 0 <= to < ROWS and 0 <= at < ROWS:
                state[:, to] = old_state[:, at]


@pytest.mark.parametrize("parents,lengths,pages,places,match", [
    ([[3, 0, 1, -1], [1, 2, 3, 0]], [21, 13], {}, {}, None),
    ([[4, 0, 1, 2], [1, 99, 3, 0]], [21, 13], {}, {}, "position"),
    ([[1, 2, 3, 0], [3, 3, 3, 0]], [21, 13], {1: -1}, {}, "block-table"),
    ([[1, 2, 3, 0], [3, 3, 3, 0]], [21, 13], {7: PAGES}, {}, "block-table"),
    ([[1, 2, 3, 0], [1, 1, 0, 0]], [21, 13], {}, {2: -1, 5: ROWS}, "position"),
    ([[1, 7, 3, 0], [1, 1, 0, 0]], [21, 13], {0: -5, 4: 1 << 30}, {3: 1 << 30}, "position.*|block-table.*"),
    ([[1, 2, 3, 0], [1, 1, 0, 0]], [-4, 16], {}, {}, None),
    ([[1, 2, 3, 0], [1, 1, 0, 0]], [24, 29], {}, {}, "position"),  # the table has three pages: the page behind 24 slots is not needed, that of 29 is not there
])
def test_what_stays_and_what_moves(parents, lengths, pages, places, match):
    random = torch.Generator().manual_seed(len(str(parents)) + sum(lengths))
    table = torch.randperm(PAGES, generator=random)[:24].to(torch.int32).view(8, 3)
    for beam, page in pages.items():
        table[beam, max(0, lengths[beam // 4]) // PAGE] = page
    rows = torch.randperm(ROWS, generator=random)[:8].to(torch.int32)
    for beam, place in places.items():
        rows[beam] = place
    cache, state = torch.randn(2, PAGES, 3, PAGE, 16, generator=random), torch.randn(3, ROWS, 37, generator=random)
    parents, lengths = torch.tensor(parents, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
    there = [x.cuda() for x in (parents, lengths, table, cache, state, rows)]
    beam_reorder(there[0], there[1], there[2], [there[3]], [there[4]], state_rows=there[5])
    if match:
        with pytest.raises(ops.KernelError, match=match):
            ops.raise_on_status(there[0].device)
    ops.raise_on_status(there[0].device)
    expected(parents, lengths, table, cache, state, rows)
    for got, want in zip(there[2:], (table, cache, state, rows)):
        assert torch.equal(got.cpu(), want)
