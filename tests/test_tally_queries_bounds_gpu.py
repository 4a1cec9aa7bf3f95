"""Queries and slots beyond the bounds that a call of ``tally_queries`` gives, and rows that are not there: they are left out and reported, and what remains sees what it would see without the bounds.

Tolerances as in test_tally_queries_edges_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_tally_gpu import close, pages_of, queries, records
from test_tally_queries_edges_gpu import given, ints

from hyperion_b200 import ops
from hyperion_b200.ops.tally import new_tally, tally_queries

pytestmark = pytest.mark.gpu


def check(starts, lengths, most, longest, *, heads=14, kv=2, dim=64, rows=40, held=300):
    """Request r has the rows ``starts[r]`` to ``starts[r + 1] - 1`` of ``rows`` rows; every request's pages hold ``held`` slots."""
    requests = len(lengths)
    cache, table, random = pages_of([held] * requests, kv, dim, 16, seed=held + rows, slack=0)
    q, tally = queries(random, rows, heads * dim), new_tally(requests, kv, table.shape[1] * 16)
    tally_queries(q, heads, cache, table, ints(starts), ints(lengths), tally, dim ** -0.5, most=most, longest=longest)
    wrong = False
    for r, length in enumerate(lengths):
        first, end = starts[r: r + 2]
        wrong |= not (0 <= first <= end <= rows and end - first <= most and 0 <= length <= longest)
        sees, at = [], []
        for row in range(max(0, first), min(end, rows)):  # of query row - first
            if len(at) < most:
                at.append(row)
                sees.append(max(0, min(length - (end - first) + row - first + 1, length, longest)))
        keys, _ = records(cache, table, r, held)
        want, off = given(q[at].view(len(at), heads, dim), keys, sees, dim ** -0.5)
        close(tally.weights[r, :, :held], want, off)
        assert bool((tally.weights[r, :, max(0, min(length, longest)):] == 0).all())
    if wrong:
        with pytest.raises(ops.KernelError, match="position"):
            ops.raise_on_status(q.device)
    ops.raise_on_status(q.device)


@pytest.mark.parametrize("starts,lengths,most", [([0, 10], [100], 8), ([0, 3, 40], [50, 300], 20), ([0, 37, 40], [290, 3], 36)])
def test_more_queries_than_most(starts, lengths, most):
    check(starts, lengths, most, 300)


@pytest.mark.parametrize("starts,lengths,longest", [([0, 10], [100], 60), ([0, 40], [200], 180), ([0, 20, 40], [300, 70], 64), ([0, 20, 40], [130, 128], 128), ([0, 40], [290], 1)])
def test_longer_than_longest(starts, lengths, longest):
    check(starts, lengths, 40, longest)


def test_both_at_once():
    check([0, 40], [200], 30, 170)


@pytest.mark.parametrize("starts", [[0, 45], [30, 47], [-3, 20], [-5, 44], [20, 10], [41, 44], [-9, -2], [-2 ** 31, 2 ** 31 - 1], [-90, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31]])
def test_rows_that_are_not_there(starts):
    check(starts, [90], 64, 300)


@pytest.mark.parametrize("length", [-7, -2 ** 31, 2 ** 31 - 1])
def test_lengths_of_none(length):
    check([0, 4, 20], [length, 50], 40, 300)


def test_a_few_queries_of_long_contexts():
    """Queries of one tile, which tiles of slots pass."""
    check([0, 5, 9], [5000, 20000], 4, 14000, heads=24, kv=1, held=20000)


def test_bounds_that_hold_are_not_reported():
    check([0, 30, 40], [300, 10], 30, 300)
