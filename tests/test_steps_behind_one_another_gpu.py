"""Steps of a beam search launched one right behind the other, no other kernel between them: each reads the tables, pages and tallies that the one before has just changed in place, and everything is, to the bit, what it
is where the device is waited for between them."""
from __future__ import annotations

import pytest
import torch
from test_tally_gpu import queries

from hyperion_b200 import ops
from hyperion_b200.ops import Tally

pytestmark = pytest.mark.gpu


def same(gots, wants):
    for got, want in zip(gots, wants):
        kind = {2: torch.int16, 4: torch.int32}[got.element_size()]
        assert torch.equal(got.view(kind), want.view(kind))


def wait(waits):
    if waits:
        torch.cuda.synchronize()


@pytest.mark.parametrize("groups,beams,heads,kv,dim,page,length", [(16, 8, 8, 2, 64, 8, 500), (1, 4, 14, 2, 64, 16, 1000), (40, 5, 28, 4, 128, 16, 131), (3, 32, 4, 4, 128, 8, 77), (2, 4, 20, 1, 128, 32, 5000)])
def test_reordered_tables_are_read_by_the_next_kernel(groups, beams, heads, kv, dim, page, length):
    random, rows, steps = torch.Generator().manual_seed(beams), groups * beams, 24
    blocks = length // page + 1
    pages = rows * blocks
    table = torch.randperm(pages, generator=random).to(torch.int32).view(rows, blocks).cuda()
    cache = torch.randn(pages, 2, kv, page, dim, generator=random).to(torch.bfloat16).cuda()
    q, q_many = queries(random, rows, heads * dim), queries(random, 2 * rows, heads * dim)
    parents = torch.randint(0, beams, (steps, groups, beams), generator=random).to(torch.int32).cuda()
    held = torch.full((groups,), length, dtype=torch.int32).cuda()
    lengths = held.repeat_interleave(beams)
    starts = torch.arange(0, 2 * rows + 1, 2, dtype=torch.int32).cuda()
    weights = torch.rand(rows, kv, blocks * page, generator=random).cuda()
    keep = max(1, length - 1 - length // 3)

    def state():
        x = [table.clone(), cache.clone(), Tally(weights.clone(), torch.arange(blocks * page, dtype=torch.int32, device="cuda").expand(weights.shape).contiguous())]
        torch.cuda.synchronize()
        return x

    def go(waits):
        tables, pool, tally = state()
        mixed = pool.view(1, pages, 2 * kv, page, dim)
        outs = [torch.empty(rows, heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(steps)]
        torch.cuda.synchronize()
        for i in range(steps):
            ops.beam_reorder(parents[i], held, tables, [mixed], [tally.weights.view(1, rows, -1), tally.positions.view(1, rows, -1)])
            wait(waits)
            if i % 3 == 2:
                ops.tally_queries(q_many, heads, pool, tables, starts, lengths, tally, dim ** -0.5, most=2)
                wait(waits)
            ops.attention_tallied(q, heads, pool, tables, lengths, lengths, tally, dim ** -0.5, out=outs[i])
            wait(waits)
        torch.cuda.synchronize()
        return [*outs, tables, pool, *tally]

    same(go(False), go(True))
    ops.raise_on_status(q.device)

    def cut(waits):
        _, pool, tally = state()
        own = torch.arange(pages, dtype=torch.int32, device="cuda").view(rows, blocks)
        results, now = [], lengths
        torch.cuda.synchronize()
        for budget in (length, keep, keep - keep // 4, max(1, keep // 2), 1):
            now = ops.evict(pool, own, now, now, tally, budget, first=1, recent=2)
            wait(waits)
            results.append(ops.attention_tallied(q, heads, pool, own, now, now, tally, dim ** -0.5))
            wait(waits)
        torch.cuda.synchronize()
        return [*results, pool, *tally]

    same(cut(False), cut(True))
    ops.raise_on_status(q.device)
