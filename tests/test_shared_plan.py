"""The host's plan of attention behind shared positions: every (token, key) pair that has to be seen is in exactly one item, and pieces are numbered without gaps."""
from __future__ import annotations

import numpy as np
import pytest

from hyperion_b200.ops import KernelError, plan_shared


def items_of(plan):
    flat = plan.data.numpy()
    n = (plan.strips + plan.tiles) * 6
    return flat[:n].reshape(-1, 6), flat[n: n + plan.tokens], flat[n + plan.tokens: n + 2 * plan.tokens + 1]


def covered(counts, lengths, heads, kv, groups, sms):
    plan = plan_shared(counts, lengths, heads, kv, 64, shared=groups, device="cpu", sms=sms)
    items, last, starts = items_of(plan)
    shared = np.zeros(len(counts), dtype=int)
    for first, n, positions in groups:
        shared[first: first + n] = positions
    owner = np.repeat(np.arange(len(counts)), counts)
    seen, pieces = [set() for _ in owner], [[] for _ in owner]
    for i, (tok, n, row, low, high, number) in enumerate(items):
        rows = plan.strip_rows if i < plan.strips else 256
        assert n >= 1 and high > low and n * min(rows, heads // kv) <= rows
        for t in range(tok, tok + n):
            assert row == owner[t] or (high <= shared[owner[t]] == shared[row])  # another request's table for shared positions only
            assert not seen[t] & set(range(low, high))
            seen[t] |= set(range(low, high))
            pieces[t].append(number)
    first = np.cumsum(np.concatenate([[0], counts]))
    for t, r in enumerate(owner):
        assert last[t] == lengths[r] - counts[r] + (t - first[r])
        assert seen[t] == (set(range(lengths[r])) if lengths[r] else set())
        assert sorted(pieces[t]) == list(range(starts[t + 1] - starts[t]))
    assert plan.pieces == (starts[-1] if len(owner) else 0) and plan.joined == any(len(p) != 1 for p in pieces)
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


def test_a_prompt_s_portion_and_a_step_of_nothing():
    covered([70], [500], 14, 2, [], 148)
    covered([0, 0], [5, 0], 14, 2, [(0, 2, 3)], 148)
    covered([], [], 14, 2, [], 148)


def test_the_device_is_filled_but_not_cut_to_pieces():
    plan = covered([1], [20000], 28, 4, [], 148)
    assert 148 <= plan.strips * 4 <= 3 * 148
    assert covered([1], [190], 28, 4, [], 148).strips == 1


def test_refusals():
    good = dict(counts=[1, 1], lengths=[9, 9], heads=4, kv_heads=2, head_dim=64, device="cpu", sms=148)
    for bad in (dict(counts=[1]), dict(counts=[1, -1]), dict(lengths=[9, -2]), dict(heads=5), dict(kv_heads=0), dict(lengths=[2**31, 9]), dict(shared=[(0, 3, 4)]), dict(shared=[(0, 2, 4), (1, 1, 4)]),
                dict(shared=[(1, 1, 4), (0, 1, 4)]), dict(shared=[(0, 2, 9)]), dict(shared=[(0, 1, -1)])):
        with pytest.raises(KernelError):
            plan_shared(**{**good, **bad})
