"""The weights of many queries where keys are infinite, against the formulas in 64 bits.

Tolerances: as derived in test_tally_gpu.py for a softmax weight; a slot's sum over rows is added up in float, 32 of a tile of 128 rows one behind the other, 4 partial sums, over tiles with what is lost, and by up to 16
blocks: less than 64 additions that round, each by 2^-24 of the sum."""
from __future__ import annotations

import pytest
import torch
from test_tally_gpu import LOG2E, close, pages_of, queries, records

from hyperion_b200 import ops
from hyperion_b200.ops.native import sm_count
from hyperion_b200.ops.tally import new_tally, tally_queries

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def given(q, keys, sees, scale):
    """What queries [n, heads, d] of which query i sees the first ``sees[i]`` slots give the keys [kv, slots, d], and what that may be off by."""
    (kv, slots, dim), (n, heads, _) = keys.shape, q.shape
    weights, off = torch.zeros(kv, slots, dtype=torch.float64, device="cuda"), torch.zeros(kv, slots, dtype=torch.float64, device="cuda")
    finite = keys.nan_to_num(neginf=0.0)
    for i in range(n):
        if sees[i] <= 0:
            continue
        x = q[i].double().view(kv, heads // kv, dim)
        p = torch.softmax(torch.einsum("kgd,knd->kgn", x, keys[:, : sees[i]]) * scale, -1)
        size = torch.einsum("kgd,knd->kgn", x.abs(), finite[:, : sees[i]].abs()).amax(-1, keepdim=True) * scale * LOG2E
        e = 2 * (0.6931471805599453 * 2.0 ** -22 * ((dim / 16 + 4) * size + 20) + 2.0 ** -21) + 64 * 2.0 ** -24
        weights[:, : sees[i]] += p.sum(1)
        off[:, : sees[i]] += (p * e).sum(1)
    return weights, off + weights * 64 * 2.0 ** -24 + 2.0 ** -120


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (28, 4, 128), (24, 1, 128), (40, 1, 64), (65, 1, 64), (100, 1, 64), (16, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("few", [False, True])  # tiles of queries pass the slots; queries of one tile, which the slots pass
def test_keys_of_negative_infinity_are_given_nothing(heads, kv, dim, few):
    """By queries that are positive, so that their scores are -infinity.  A tile of queries has 128 // group tokens; where the group does not divide 128 it has rows that are no one's, and tiles of slots are seen in full here."""
    per_tile = 128 // (heads // kv)
    count, length = (per_tile, (sm_count() // kv + 2) * 128 + 50) if few else (3 * per_tile + 1, 3 * per_tile + 700)
    cache, table, random = pages_of([length], kv, dim, 16, seed=heads)
    q = queries(random, count, heads * dim).abs() + 0.125
    lost = sorted({0, 5, 127, 128, 300, 301, 600, length - count - 1, length - 1})
    for slot in lost:
        cache[table[0, slot // 16], 0, :, slot % 16, 7] = float("-inf")
    tally = new_tally(1, kv, table.shape[1] * 16)
    tally_queries(q, heads, cache, table, ints([0, count]), ints([length]), tally, dim ** -0.5, most=count)
    ops.raise_on_status(q.device)
    keys, _ = records(cache, table, 0, length)
    want, off = given(q.view(count, heads, dim), keys, [length - count + i + 1 for i in range(count)], dim ** -0.5)
    assert bool((want[:, lost] == 0).all()) and bool((tally.weights[0][:, lost] == 0).all())
    assert not tally.weights.isnan().any()
    close(tally.weights[0, :, :length], want, off)


@pytest.mark.parametrize("heads,kv,count,length", [(8, 1, 500, 500), (14, 2, 300, 300), (8, 1, 450, 640), (24, 1, 90, 512)])
def test_clusters_of_sixteen_blocks(heads, kv, count, length):
    """Few tiles of slots (of 128) and many of queries (of 128 // group): with less than 0.7 blocks a multiprocessor, sixteen share a tile of slots."""
    tiles, per_tile = -(-length // 128) * kv, 128 // (heads // kv)
    assert 16 * tiles <= 0.7 * sm_count() and count > 15 * per_tile
    cache, table, random = pages_of([length], kv, 64, 16, seed=count)
    q, tally = queries(random, count, heads * 64), new_tally(1, kv, table.shape[1] * 16)
    tally_queries(q, heads, cache, table, ints([0, count]), ints([length]), tally, 0.125, most=count)
    ops.raise_on_status(q.device)
    keys, _ = records(cache, table, 0, length)
    want, off = given(q.view(count, heads, 64), keys, [length - count + i + 1 for i in range(count)], 0.125)
    close(tally.weights[0, :, :length], want, off)
    assert bool((tally.weights[0, :, length:] == 0).all())
