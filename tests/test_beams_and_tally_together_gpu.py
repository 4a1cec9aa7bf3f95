"""Calls of the operators of beams and of caches of a fixed budget as a server makes them: captured and replayed with other lengths, on other streams, from threads on one stream, again with the same result."""
from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor
from threading import Barrier

import pytest
import torch
from test_beams_gpu import some_logits
from test_tally_gpu import pages_of, queries

from hyperion_b200 import ops
from hyperion_b200.ops import Tally
from hyperion_b200.sampling import beam_select

pytestmark = pytest.mark.gpu
THREADS = 4


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Work:
    """All five operators on data of their own; ``lengths`` and the rest are tensors, so that a captured call can go on with others."""

    def __init__(self, seed, most=3000, requests=6):
        self.heads, self.kv, self.dim = 8, 2, 64
        self.lengths_list = [(most - 377 * i - 11 * seed) % most + 1 for i in range(requests)]
        self.cache, self.table, random = pages_of([most] * requests, self.kv, self.dim, 16, seed=seed, slack=0)
        self.q, self.many = queries(random, requests, 8 * 64), queries(random, 40, 8 * 64)
        self.lengths, self.starts = ints(self.lengths_list), ints([0, 3, 3, 40, 40, 40, 40])
        self.capacity = self.table.shape[1] * 16
        self.weights = torch.rand(requests, self.kv, self.capacity, generator=random).cuda()
        self.logits, self.scores = some_logits(2, 3, 20001, seed=seed)
        self.tally = Tally(torch.empty_like(self.weights), torch.empty(self.weights.shape, dtype=torch.int32, device="cuda"))
        self.after = Tally(torch.empty_like(self.weights), torch.empty_like(self.tally.positions))
        self.pages = self.cache.clone()
        self.blocks = self.table.clone()

    def run(self):
        positions = torch.arange(self.capacity, dtype=torch.int32, device="cuda")
        self.tally.weights.copy_(self.weights), self.tally.positions.copy_(positions.expand(self.weights.shape))
        self.pages.copy_(self.cache), self.blocks.copy_(self.table)
        ops.tally_queries(self.many, self.heads, self.pages, self.table, self.starts, self.lengths, self.tally, 0.1, most=37)
        out = ops.attention_tallied(self.q, self.heads, self.pages, self.table, self.lengths, self.lengths, self.tally, 0.1)
        left = ops.evict(self.pages, self.table, self.lengths, self.lengths - 1, self.tally, 900, first=4, recent=50, out=self.after)
        choice = beam_select(self.logits, self.scores, 3)
        ops.beam_reorder(choice.parents, left[:2].contiguous(), self.blocks, [self.pages.view(1, -1, 2 * self.kv, 16, self.dim)], [self.after.weights.view(1, 6, -1)])
        return [out.clone(), self.tally.weights.clone(), self.after.weights.clone(), self.after.positions.clone(), left.clone(), choice.parents.clone(), choice.tokens.clone(), choice.scores.clone(),
                self.pages.view(torch.int16).clone(), self.blocks.clone()]


def same(got, want):
    return all(torch.equal(a.view(torch.int32) if a.dtype is torch.float32 else a, b.view(torch.int32) if b.dtype is torch.float32 else b) for a, b in zip(got, want))


def test_again_with_the_same_result_to_the_bit():
    work = Work(0)
    want = work.run()
    for _ in range(20):
        assert same(work.run(), want)
    ops.raise_on_status(work.q.device)


def test_captured_and_replayed_with_other_lengths():
    work = Work(1)
    shorter = ints([5, 1, 2999, 40, 900, 901])
    first = work.lengths.clone()
    want_first = work.run()
    work.lengths.copy_(shorter)
    want_shorter = work.run()
    work.lengths.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work.run()
    for lengths, want in ((first, want_first), (shorter, want_shorter), (first, want_first)):
        work.lengths.copy_(lengths)
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, want)
    ops.raise_on_status(work.q.device)


def test_two_captured_graphs_side_by_side():
    works = [Work(2), Work(3)]
    wants = [work.run() for work in works]
    graphs, gots, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for work in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gots.append(work.run())
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        assert same(got, want)
    ops.raise_on_status(works[0].q.device)


def test_on_streams_of_their_own():
    works = [Work(4), Work(5), Work(6)]
    wants = [work.run() for work in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    gots = [None] * len(works)
    for _ in range(5):
        for i, (work, stream) in enumerate(zip(works, streams)):
            with torch.cuda.stream(stream):
                gots[i] = work.run()
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        assert same(got, want)
    ops.raise_on_status(works[0].q.device)


def test_threads_on_one_stream():
    works = [Work(7 + i, most=1500) for i in range(THREADS)]
    wants = [work.run() for work in works]
    torch.cuda.synchronize()
    together = Barrier(THREADS)

    def go(i):
        together.wait(10)
        return [works[i].run() for _ in range(30)]

    with ThreadPoolExecutor(THREADS) as pool:
        answers = list(pool.map(go, range(THREADS)))
    torch.cuda.synchronize()
    ops.raise_on_status(works[0].q.device)
    for got, want in zip(answers, wants):
        assert all(same(answer, want) for answer in got)


def test_nothing_to_do():
    """No requests, no groups, no queries, requests without slots: nothing is launched or written."""
    cache, table, random = pages_of([40, 0], 2, 64, 16, seed=1)
    tally = ops.new_tally(0, 2, 48)
    assert ops.attention_tallied(torch.empty(0, 512, dtype=torch.bfloat16, device="cuda"), 8, cache, table, ints([]), ints([]), tally, 0.1).shape == (0, 512)
    ops.tally_queries(torch.empty(0, 512, dtype=torch.bfloat16, device="cuda"), 8, cache, table, ints([0]), ints([]), tally, 0.1, most=0)
    assert ops.evict(cache, table, ints([]), ints([]), tally, 4).shape == (0,)
    assert beam_select(torch.empty(0, 100, device="cuda"), torch.empty(0, 4, device="cuda"), 4).tokens.shape == (0, 4)
    ops.beam_reorder(torch.empty(0, 4, dtype=torch.int32, device="cuda"), ints([]), None, [], [torch.empty(2, 0, 5, device="cuda")])
    two = ops.new_tally(2, 2, 48)
    before = two.weights.clone()
    out = ops.attention_tallied(queries(random, 2, 512), 8, cache, table, ints([0, 0]), ints([7, 7]), two, 0.1)
    assert bool((out == 0).all()) and torch.equal(two.weights, before)
    out = ops.attention_tallied(queries(random, 2, 512), 8, cache, table, ints([0, 0]), ints([7, 7]), two, 0.1, longest=0)
    assert bool((out == 0).all())
    ops.tally_queries(queries(random, 4, 512), 8, cache, table, ints([0, 2, 4]), ints([0, 0]), two, 0.1, most=2)
    assert torch.equal(two.weights, before)
    given = cache.clone()
    assert ops.evict(cache, table, ints([0, 0]), ints([0, 0]), two, 4).tolist() == [0, 0]
    assert torch.equal(given.view(torch.int16), cache.view(torch.int16)) and torch.equal(two.weights, before) and two.positions[0, 0].tolist() == list(range(48))
    ops.raise_on_status(cache.device)
