"""Eviction of what weighs least, against the rule slot by slot: records, weights and positions are moved, so everything is equal to the bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops.tally import Tally, evict

pytestmark = pytest.mark.gpu


def bits(x):
    return x.contiguous().view(torch.uint8).cpu().numpy().copy()


def expected(cache, table, lengths, newest, weights, positions, keep, first, recent, separate):
    """cache [layers, pages, 2, kv, page, bytes]; the rest as it goes into evict; all numpy.  In place, slots behind a request stay as they were."""
    cache, out_w, out_p = cache.copy(), np.zeros_like(weights), np.full_like(positions, -1)
    if not separate:
        for r, n in enumerate(lengths):
            out_w[:, r, :, n:], out_p[:, r, :, n:] = weights[:, r, :, n:], positions[:, r, :, n:]
    page = cache.shape[4]
    for layer in range(weights.shape[0]):
        for r, n in enumerate(lengths):
            for h in range(weights.shape[2]):
                w, p = weights[layer, r, h], positions[layer, r, h]
                if n <= keep:
                    out_w[layer, r, h, :n], out_p[layer, r, h, :n] = w[:n], p[:n]
                    continue
                rank = np.where(np.isnan(w[:n]), -np.inf, w[:n]).astype(np.float64)
                rank[(p[:n] < first) | (p[:n].astype(np.int64) > int(newest[r]) - recent)] = np.inf
                stays = np.zeros(n, dtype=bool)
                stays[np.lexsort((np.arange(n), -rank))[:keep]] = True
                movers, holes = [s for s in range(keep, n) if stays[s]], [s for s in range(keep) if not stays[s]]
                assert len(movers) == len(holes)
                out_w[layer, r, h, :keep], out_p[layer, r, h, :keep] = w[:keep], p[:keep]
                for s, d in zip(movers, holes):
                    cache[layer, table[r, d // page], :, h, d % page] = cache[layer, table[r, s // page], :, h, s % page]
                    out_w[layer, r, h, d], out_p[layer, r, h, d] = w[s], p[s]
    return np.minimum(lengths, keep), cache, out_w, out_p


def run(lengths, *, layers=1, kv=2, dim=64, page=16, keep=10, first=0, recent=0, dtype=torch.bfloat16, seed=0, spread=None, change=None, separate=False, extra=0, longest=None, flat=False):
    random = np.random.default_rng(seed)
    blocks = -(-max(max(lengths), 1) // page) + 1
    pages, capacity = len(lengths) * blocks + 2, blocks * page + extra
    table = random.permutation(pages)[: len(lengths) * blocks].reshape(len(lengths), blocks).astype(np.int32)
    given = random.integers(0, 256, (layers, pages, 2, kv, page, dim * torch.empty(0, dtype=dtype).element_size()), dtype=np.uint8)
    shape = (layers, len(lengths), kv, capacity)
    weights = random.standard_exponential(shape).astype(np.float32)
    if spread is not None:
        weights = (np.floor(weights * spread) / spread).astype(np.float32)  # many equal ones
    positions = np.argsort(random.random(shape), axis=-1).astype(np.int32)
    newest = positions.max((0, 2, 3)).astype(np.int32)
    if change:
        change(weights, positions)
    cache, tally = torch.from_numpy(given).cuda().view(dtype), Tally(torch.from_numpy(weights.copy()).cuda(), torch.from_numpy(positions.copy()).cuda())
    if flat:
        cache, tally = cache[0], Tally(tally.weights[0], tally.positions[0])
    out = Tally(torch.full_like(tally.weights, 3.0), torch.full_like(tally.positions, 3)) if separate else None
    left = evict(cache, torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(newest).cuda(), tally, keep, first=first, recent=recent, out=out, longest=longest)
    ops.raise_on_status(cache.device)
    want_left, want_cache, want_w, want_p = expected(given, table, np.array(lengths), newest, weights, positions, keep, first, recent, separate)
    to = out if separate else tally
    assert left.tolist() == want_left.tolist()
    assert np.array_equal(to.positions.cpu().numpy().reshape(want_p.shape), want_p)
    assert np.array_equal(to.weights.cpu().numpy().reshape(want_w.shape), want_w, equal_nan=True)
    assert np.array_equal(bits(cache).reshape(want_cache.shape), want_cache)
    if separate:
        assert np.array_equal(tally.weights.cpu().numpy().reshape(shape), weights, equal_nan=True) and np.array_equal(tally.positions.cpu().numpy().reshape(shape), positions)


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("lengths,keep", [([1], 1), ([2], 1), ([65], 64), ([100, 10, 0, 37], 10), ([1500], 700), ([1025, 1024, 1023], 1024), ([3000, 5], 1), ([2500], 2499), ([2049], 2000)])
def test_lengths(lengths, keep, separate):
    run(lengths, keep=keep, separate=separate, seed=keep)


@pytest.mark.parametrize("layers,kv,dim,page,dtype", [(3, 4, 128, 64, torch.bfloat16), (2, 1, 64, 8, torch.float32), (1, 3, 16, 1, torch.float8_e4m3fn), (2, 8, 256, 32, torch.float16), (1, 2, 96, 16, torch.bfloat16)])
def test_layouts(layers, kv, dim, page, dtype):
    run([300, 120], layers=layers, kv=kv, dim=dim, page=page, dtype=dtype, keep=77, first=4, recent=20, extra=3)


def test_without_layers():
    run([300, 120], kv=3, keep=50, flat=True)
    run([300, 120], kv=3, keep=50, flat=True, separate=True)


@pytest.mark.parametrize("first,recent", [(0, 0), (4, 0), (0, 1), (5, 60), (40, 80), (1000, 0), (0, 5000)])
def test_first_and_latest_positions_stay(first, recent):
    run([400, 90], layers=2, keep=64, first=first, recent=recent)


@pytest.mark.parametrize("spread", [0.001, 1, 4])
def test_of_equal_weights_the_lowest_slots_stay(spread):
    run([2300, 700], keep=333, spread=spread, separate=spread == 1)


def test_weights_of_all_kinds():
    def change(weights, positions):
        flat = weights.reshape(-1)
        flat[::3] *= -1
        flat[::7] = np.nan
        flat[1::11] = np.inf
        flat[2::11] = -np.inf
        flat[3::13] = -0.0
        flat[4::13] = 0.0
        flat[5::17] = np.float32(1e-42)
    for keep in (50, 300, 600, 700):
        run([777, 900], keep=keep, change=change, seed=keep, separate=keep == 300)


@pytest.mark.parametrize("length,keep,layers,kv", [(300000, 200, 1, 1), (40001, 9000, 1, 2), (9001, 9000, 2, 1), (33000, 1, 1, 1), (70000, 69000, 1, 1)])
def test_long_requests(length, keep, layers, kv):
    run([length], layers=layers, kv=kv, dim=16, page=64, keep=keep, first=4, recent=min(keep, 64))


def test_more_slots_than_a_cluster_holds():
    run([450001, 5000], kv=1, dim=8, page=64, keep=1000, first=4, recent=64, separate=True)


@pytest.mark.parametrize("separate", [False, True])
def test_records_that_a_second_kernel_moves(separate):
    run([9000, 200], kv=2, dim=256, page=64, dtype=torch.float32, keep=4000, separate=separate)


@pytest.mark.parametrize("kv,layers", [(1, 1), (8, 4), (8, 20)])  # clusters of many blocks, of some, of one
def test_equal_weights_across_the_blocks_of_a_cluster(kv, layers):
    for spread in (0.001, 2):
        run([12000], kv=kv, layers=layers, dim=8, page=64, keep=5000, first=3, recent=100, spread=spread)


def test_a_bound_on_the_lengths():
    run([300, 120], keep=40, longest=300)
    run([30, 12], keep=40, longest=30)


def test_again_and_again_to_the_same_budget():
    """A conversation at its budget: each token enters, the least of all leaves; what is left are the heaviest of all that ever came."""
    random, keep, page = np.random.default_rng(1), 24, 8
    cache = torch.zeros(1, 5, 2, 1, page, 16, dtype=torch.bfloat16, device="cuda")
    table, capacity = torch.tensor([[4, 0, 3, 1]], dtype=torch.int32, device="cuda"), 32
    tally = Tally(torch.zeros(1, 1, 1, capacity, device="cuda"), torch.full((1, 1, 1, capacity), -1, dtype=torch.int32, device="cuda"))
    came, length = [], 0
    for position in range(200):
        weight = float(np.float32(random.standard_exponential()))
        came.append(weight)
        cache[0, table[0, length // page], :, 0, length % page] = position % 256
        tally.weights[0, 0, 0, length], tally.positions[0, 0, 0, length] = weight, position
        length += 1
        one = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
        length = int(evict(cache, table, one(length), one(position), tally, keep).item())
        assert length == min(position + 1, keep)
    ops.raise_on_status(cache.device)
    held = sorted(tally.positions[0, 0, 0, :keep].tolist())
    assert held == sorted(np.argsort(-np.array(came), kind="stable")[:keep].tolist())
    for slot in range(keep):
        position = int(tally.positions[0, 0, 0, slot])
        assert float(tally.weights[0, 0, 0, slot]) == came[position]
        assert bool((cache[0, table[0, slot // page], :, 0, slot % page] == position % 256).all())


def test_what_is_not_there_is_reported():
    cache = torch.zeros(4, 2, 1, 8, 64, dtype=torch.bfloat16, device="cuda")
    one = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    def tally():
        return Tally(torch.arange(24, device="cuda", dtype=torch.float32).view(1, 1, 24), torch.arange(24, device="cuda", dtype=torch.int32).view(1, 1, 24).contiguous())
    for table in ([[0, -1, 2]], [[9, 1, 2]]):
        evict(cache, torch.tensor(table, dtype=torch.int32, device="cuda"), one(20), one(19), tally(), 8)
        with pytest.raises(ops.KernelError, match="block-table entry"):
            ops.raise_on_status(cache.device)
    left = evict(cache, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), one(21), one(20), tally(), 8, longest=20)
    assert left.tolist() == [8]
    with pytest.raises(ops.KernelError, match="position"):
        ops.raise_on_status(cache.device)
