"""Calls of several kernels that keep something in scratch memory between them, from threads that launch on the same stream: another thread's launches may come between two of one call."""
from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor
from threading import Barrier

import pytest
import torch
from test_shared_attention_gpu import step
from test_verify_drafts_gpu import case

from hyperion_b200 import ops
from hyperion_b200.ops.native import KEPT_SCRATCH, scratch
from hyperion_b200.ops.shared import attention_shared, plan_shared
from hyperion_b200.sampling import verify_drafts

pytestmark = pytest.mark.gpu
THREADS = 4


def test_a_thread_has_memory_of_its_own():
    together, device = Barrier(THREADS), torch.device("cuda", torch.cuda.current_device())

    def work(_):
        first = [scratch(device, stream, 1000) for stream in (0, 1)]
        again = scratch(device, 0, 2000)
        together.wait(10)  # all threads are there, so that every one of them has its own
        return [address for address, _ in first], again[0]

    with ThreadPoolExecutor(THREADS) as pool:
        answers = list(pool.map(work, range(THREADS)))
    assert len({address for first, _ in answers for address in first}) == 2 * THREADS  # per thread and stream
    assert all(first[0] == again for first, again in answers)  # kept for the next call


def pieces(seed, bits):
    """One long request whose pieces go through memory."""
    q, cache, table = step([1], [9000 + 200 * seed], 14, 2, 64, 16, bits, seed=seed)
    plan = plan_shared([1], [9000 + 200 * seed], 14, 2, 64)
    assert plan.joined and not plan.together and not plan.tile_blocks
    return lambda: attention_shared(q, 14, cache, table, plan, 0.1)


def tiles(seed, bits):
    """Requests behind shared positions: operands (of 8-bit records), tiles, strips beside them, and the joining."""
    counts, lengths, groups = [1] * 30, [700 + 3 * seed + r for r in range(30)], [(0, 30, 600 + seed)]
    q, cache, table = step(counts, lengths, 8, 2, 64, 16, bits, groups, seed=seed)
    plan = plan_shared(counts, lengths, 8, 2, 64, shared=groups)
    assert plan.joined and not plan.together and plan.tile_blocks and plan.strip_blocks and plan.operand_tiles
    assert plan.pieces * 8 * 66 * 4 + plan.operand_tiles * 2 * 2 * 128 * 2 * 64 < KEPT_SCRATCH
    return lambda: attention_shared(q, 8, cache, table, plan, 0.1)


def drafts(seed, dtype):
    c = case([3, 0, 5, 2], 40001, seed, dtype)
    return lambda: torch.cat([answer.view(-1) for answer in verify_drafts(**c)])


@pytest.mark.parametrize("what", [lambda s: pieces(s, 8), lambda s: pieces(s, 16), lambda s: tiles(s, 8), lambda s: tiles(s, 16), lambda s: drafts(s, torch.float32),
                                  lambda s: (pieces, tiles, tiles, drafts)[s](s, (8, 8, 16, torch.bfloat16)[s])],
                         ids=["pieces 8", "pieces 16", "tiles 8", "tiles 16", "drafts", "all"])
def test_threads_on_one_stream(what):
    calls = [what(seed) for seed in range(THREADS)]
    want = [call() for call in calls]
    together = Barrier(THREADS)

    def work(i):
        together.wait(10)
        return [calls[i]() for _ in range(200)]

    with ThreadPoolExecutor(THREADS) as pool:
        got = list(pool.map(work, range(THREADS)))
    ops.raise_on_status(got[0][0].device)
    assert all(torch.equal(answer, expected) for answers, expected in zip(got, want) for answer in answers)
