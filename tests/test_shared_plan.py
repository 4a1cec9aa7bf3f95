"""The host's plan of attention behind shared positions: every (token, key) pair that has to be seen is in exactly one item, and pieces are numbered without gaps."""
from __future__ import annotations

import numpy as np
import pytest

from hyperion_b200.ops import KernelError, plan_shared

OWN = 1 << 30


def parts_of(plan):
    """(items of strips with their blocks, the same of tiles, last positions, first pieces, first own pieces)"""
    flat, at = plan.data.numpy(), plan.places + [plan.data.numel()]
    sizes = [at[1], plan.strip_blocks + 1, at[3] - at[2], plan.tile_blocks + 1, plan.tokens, plan.tokens + 1, plan.tokens, 4 * plan.operand_tiles]
    part = [flat[at[i]: at[i] + n] for i, n in enumerate(sizes)]
    part[0], part[2] = (items[: 7 * first[-1]] for items, first in ((part[0], part[1]), (part[2], part[3])))
    assert all(place % 4 == 0 for place in plan.places)
    walks = []
    for items, first in ((part[0], part[1]), (part[2], part[3])):
        items = items.reshape(-1, 7)
        assert first[0] == 0 and first[-1] == len(items) and (np.diff(first) > 0).all()
        walks.append((items, np.repeat(np.arange(len(first) - 1), np.diff(first))))
    return walks[0], walks[1], part[4], part[5], part[6], part[7].reshape(-1, 4)


def covered(counts, lengths, heads, kv, groups, sms):
    plan = plan_shared(counts, lengths, heads, kv, 64, shared=groups, device="cpu", sms=sms)
    strips, tiles, last, starts, own, operands = parts_of(plan)
    shared = np.zeros(len(counts), dtype=int)
    for first, n, positions in groups:
        shared[first: first + n] = positions
    owner = np.repeat(np.arange(len(counts)), counts)
    seen, pieces = [set() for _ in owner], [[] for _ in owner]
    for rows, (items, _) in ((plan.strip_rows, strips), (256, tiles)):
        for tok, n, row, low, high, number, operand in items:
            assert n >= 1 and (high > low or (plan.together and low == high == 0)) and n * min(rows, heads // kv) <= rows
            if rows == 256:  # the item's tiles stand one behind the other among the operands
                for i, at in enumerate(range(low // 128 * 128, high, 128)):
                    assert operands[operand + i][0] == row and operands[operand + i][1] == at and operands[operand + i][2] <= low and high <= operands[operand + i][3]
            for t in range(tok, tok + n):
                assert (low >= shared[row] and row == owner[t]) if number & OWN else (high <= shared[owner[t]] == shared[row])  # another request's table for shared positions only
                assert not seen[t] & set(range(low, high))
                seen[t] |= set(range(low, high))
                pieces[t].append((own if number & OWN else starts)[t] + (number & (OWN - 1)))
    first = np.cumsum(np.concatenate([[0], counts]))
    for t, r in enumerate(owner):
        assert last[t] == max(-1, lengths[r] - counts[r] + (t - first[r]))
        assert seen[t] == set(range(lengths[r]))
        assert sorted(pieces[t]) == list(range(starts[t], starts[t + 1]))
    assert plan.operand_tiles == len(operands)
    assert plan.pieces == starts[-1] and plan.joined == any(len(p) != 1 for p in pieces)
    if plan.together:  # blocks in a row have the same tokens, an item each
        same = strips[0][:, :3].reshape(-1, plan.together, 3)
        assert 2 <= plan.together <= 8 and len(tiles[0]) == 0 and (same == same[:, :1]).all() and not shared.any()
    assert (plan.strip_blocks, plan.tile_blocks) == tuple(len(np.unique(b)) for _, b in (strips, tiles))
    return plan


@pytest.mark.parametrize("sms", [1, 148])
@pytest.mark.parametrize("heads,kv", [(14, 2), (4, 4), (40, 2)])
def test_every_pair_once(heads, kv, sms):
    random = np.random.default_rng(heads + sms)
    for _ in range(30):
        requests = int(random.integers(1, 9))
        counts, shared = random.integers(0, 6, requests), np.zeros(requests, dtype=int)
        groups, at = [], 0
        while at < requests:
            n = int(random.integers(1, 4))
            if at + n <= requests and random.random() < 0.6:
                positions = int(random.integers(0, 700))
                groups.append((at, n, positions))
                shared[at: at + n] = positions
            at += n
        lengths = shared + counts + random.integers(0, 300, requests)
        lengths[(shared == 0) & (random.random(requests) < 0.2)] = 0
        covered(counts.tolist(), lengths.tolist(), heads, kv, groups, sms)


def test_portions_of_prompts_and_steps_of_nothing():
    covered([70], [500], 14, 2, [], 148)
    covered([300, 1, 20], [900, 2000, 700], 16, 4, [(0, 3, 555)], 148)
    covered([0, 0], [5, 0], 14, 2, [(0, 2, 3)], 148)
    covered([], [], 14, 2, [], 148)


@pytest.mark.parametrize("counts,lengths,groups", [([1], [20000], ()), ([1] * 64, list(range(1000, 2000, 16))[:64][: 63] + [2000], ()), ([1] * 30, [5000] * 30, ((0, 30, 4000),))])
def test_blocks_have_equal_shares(counts, lengths, groups):
    plan = plan_shared(counts, lengths, 28, 4, 128, shared=groups, device="cpu", sms=148)
    for items, block in parts_of(plan)[:2]:
        if len(items):
            keys = np.bincount(block, items[:, 4] - items[:, 3])
            assert keys.max() <= 1.5 * keys.mean() + 256 and len(keys) * 4 <= 3 * 148


def test_wide_ranges_have_operand_tiles():
    assert plan_shared([4], [500], 14, 2, 64, device="cpu", sms=148).operand_tiles == 0  # strips take records as they are
    assert plan_shared([72], [500], 14, 2, 64, device="cpu", sms=148).operand_tiles == 4
    assert plan_shared([1] * 80, [700] * 80, 14, 2, 64, shared=[(0, 80, 600)], device="cpu", sms=148).operand_tiles == 5


def test_short_ranges_stay_whole():
    plan = plan_shared([1, 1], [250, 190], 28, 4, 128, device="cpu", sms=148)
    assert plan.strip_blocks == 2 and not plan.joined and not plan.together
    plan = plan_shared([1, 1], [500, 190], 28, 4, 128, device="cpu", sms=148)  # a cluster for each
    assert plan.together == 4 and plan.strip_blocks == 8
    plan = plan_shared([1, 1, 0], [500, 190, 90], 28, 4, 128, shared=[(0, 2, 16)], device="cpu", sms=148)  # rows of two runs
    assert not plan.together and plan.joined


def test_clusters_walk_every_key():
    random = np.random.default_rng(5)
    for heads, kv in ((14, 2), (28, 4), (8, 8)):
        for _ in range(20):
            requests = int(random.integers(1, 12))
            counts = random.integers(1, 4, requests)
            lengths = counts + random.integers(0, 1500, requests)
            lengths[0] += 400
            assert covered(counts.tolist(), lengths.tolist(), heads, kv, [], 148).together


def test_refusals():
    good = dict(counts=[1, 1], lengths=[9, 9], heads=4, kv_heads=2, head_dim=64, device="cpu", sms=148)
    for bad in (dict(counts=[1]), dict(counts=[1, -1]), dict(lengths=[9, -2]), dict(heads=5), dict(kv_heads=0), dict(lengths=[2**31, 9]), dict(shared=[(0, 3, 4)]), dict(shared=[(0, 2, 4), (1, 1, 4)]),
                dict(shared=[(1, 1, 4), (0, 1, 4)]), dict(shared=[(0, 2, 9)]), dict(shared=[(0, 1, -1)]), dict(shared=[(0, 1)])):
        with pytest.raises(KernelError):
            plan_shared(**{**good, **bad})
