"""Attention that keeps its weights, and the weights of a prompt's queries, against the formulas in 64 bits.

Tolerances.  A score is a sum of d products that are exact in float, added up in d / 16 steps of the tensor cores, each off by at most 2^-22 of what it adds up (they cut, where rounding would be half of
it), then multiplied by scale * log2(e), two roundings: with S = max_j sum_i |q_i k_ji| scale log2(e), y is off by less than (d / 16 + 1) 2^-22 S.  Where queries are many, m + log2 l, which is at most S + 17 here, goes
through one more step of the tensor cores: 2^-22 (2 S + 17), and 2^-22 (S + 3) for the logarithm, the division and its three parts.  So delta = 2^-22 ((d / 16 + 4) S + 20).  A softmax weight p is 2^(y - m) / l: the power
is off by ln2 delta and 2^-22 (the hardware's), l by as much on average, so p by less than e_p = 2 (ln2 delta + 2^-21) of itself.  Sums over up to n terms in float add n 2^-24 at the most (a lane adds up few; n = 64 here).
A result is sum p v, its weights in two parts of bfloat16 (2^-16 of a weight), rounded to bfloat16 (2^-8 of it) at the end."""
from __future__ import annotations

import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops.tally import attention_tallied, new_tally, tally_queries

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


def pages_of(lengths, kv, dim, page, *, seed=0, slack=1, spare=3, size=1.0):
    """A cache whose unheld slots hold NaN, and its block table: pages in no order, `slack` more blocks than needed, -1 where a request has none."""
    random = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    width = max(max(blocks, default=0) + slack, 1)
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=random).to(torch.int32)
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    cache = torch.randn(pages, 2, kv, page, dim, generator=random) * size
    held = torch.zeros(pages, page, dtype=torch.bool)
    for r, n in enumerate(lengths):
        table[r, : blocks[r]] = order[at: at + blocks[r]]
        at += blocks[r]
        for slot in range(n):
            held[table[r, slot // page], slot % page] = True
    cache = torch.where(held[:, None, None, :, None], cache, torch.full_like(cache, float("nan")))
    return cache.to(torch.bfloat16).cuda(), table.cuda(), random


def records(cache, table, r, n):
    """Keys and values of request r in 64 bits, [2, kv, n, d]."""
    page = cache.shape[3]
    x = cache[table[r, : -(-n // page)].long()].double()
    return x.permute(1, 2, 0, 3, 4).reshape(2, cache.shape[2], -1, cache.shape[4])[:, :, :n]


def attended(q, heads, cache, table, counts, lengths, scale):
    """Per request and token: result, sum p |v|, weights [kv, slots] and what they may be off by, in 64 bits."""
    kv, dim, first, found = cache.shape[2], cache.shape[4], 0, []
    for r, (count, length) in enumerate(zip(counts, lengths)):
        k, v = records(cache, table, r, length)
        weights, off = torch.zeros(kv, length, dtype=torch.float64, device="cuda"), torch.zeros(kv, length, dtype=torch.float64, device="cuda")
        for i in range(count):
            sees = length - count + i + 1
            x = q[first + i, : heads * dim].double().view(kv, heads // kv, dim)
            if sees <= 0:
                found.append((r, torch.zeros(heads * dim, device="cuda"), torch.zeros(heads * dim, device="cuda"), 0.0))
                continue
            y = torch.einsum("kgd,knd->kgn", x, k[:, :sees]) * scale
            p = torch.softmax(y, -1)
            size = torch.einsum("kgd,knd->kgn", x.abs(), k[:, :sees].abs()).amax(-1, keepdim=True) * scale * LOG2E
            e = 2 * (0.6931471805599453 * 2.0 ** -22 * ((dim / 16 + 4) * size + 20) + 2.0 ** -21) + 64 * 2.0 ** -24
            weights[:, :sees] += p.sum(1)
            off[:, :sees] += (p * e).sum(1)
            found.append((r, (p @ v[:, :sees]).reshape(-1), ((p * (e + 2.0 ** -16)) @ v[:, :sees].abs()).reshape(-1), e.max().item()))
        first += count
        found.append((r, weights, off, None))
    return found


def close(got, want, off):
    error = (got.double() - want).abs()
    assert bool((error <= off).all()), f"off by up to {(error / off).max().item():.3f} of what it may be"


def queries(random, tokens, width, stride_more=0, size=2.0):
    x = torch.randn(tokens, width + stride_more, generator=random) * size
    return x.to(torch.bfloat16).cuda()[:, :width]


SHAPES = [(14, 2, 64, 16), (28, 4, 128, 16), (16, 16, 64, 8), (24, 1, 128, 64), (40, 1, 64, 32), (32, 8, 128, 32), (9, 1, 128, 8), (1, 1, 64, 64)]


@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
@pytest.mark.parametrize("lengths", [[1], [63, 64, 65], [0, 17, 0, 300, 1], [1000, 3, 129], [2500]])
@pytest.mark.parametrize("room", [0, 8400])  # a table that may hold more slots than a cluster of blocks keeps the scores of
def test_a_decoded_token(heads, kv, dim, page, lengths, room):
    cache, table, random = pages_of(lengths, kv, dim, page, seed=len(lengths), slack=1 + room // page)
    q = queries(random, len(lengths), heads * dim, 24)
    capacity = table.shape[1] * page
    tally = new_tally(len(lengths), kv, capacity)
    tally.weights.copy_(torch.rand(tally.weights.shape, generator=random))
    before = tally.weights.clone()
    length, newest = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.arange(len(lengths), dtype=torch.int32, device="cuda") + 70000
    out = torch.full((len(lengths), heads * dim + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    result = attention_tallied(q, heads, cache, table, length, newest, tally, dim ** -0.5, out=out)
    ops.raise_on_status(q.device)
    assert result is out and bool((out[:, heads * dim:] == 7).all())
    counts = [1] * len(lengths)
    for r, want, off, e in attended(q, heads, cache, table, counts, lengths, dim ** -0.5):
        if e is not None:
            close(out[r, : heads * dim], want, off + want.abs() * 2.0 ** -8)
            continue
        n = lengths[r]
        want = want + torch.where(torch.arange(n, device="cuda") == n - 1, 0.0, before[r, :, :n].double())
        close(tally.weights[r, :, :n], want, off + want * 2.0 ** -23)
        assert torch.equal(tally.weights[r, :, n:], before[r, :, n:])
        where = torch.arange(capacity, device="cuda", dtype=torch.int32)
        if n:
            where[n - 1] = newest[r]
        assert torch.equal(tally.positions[r], where.expand(kv, -1))


@pytest.mark.parametrize("bound", [None, 8300])
@pytest.mark.parametrize("heads,kv", [(14, 2), (20, 2)])
def test_many_requests_of_all_lengths_and_a_bound_on_them(heads, kv, bound):
    dim, page = 64, 16
    lengths = [(37 * i) % 700 for i in range(90)]
    cache, table, random = pages_of(lengths, kv, dim, page, seed=4, slack=0 if bound is None else 500)
    q = queries(random, len(lengths), heads * dim)
    tally = new_tally(len(lengths), kv, bound or 701)
    out = attention_tallied(q, heads, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.zeros(len(lengths), dtype=torch.int32, device="cuda"), tally, 0.1, longest=bound or max(lengths))
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, [1] * len(lengths), lengths, 0.1):
        if e is not None:
            close(out[r], want, off + want.abs() * 2.0 ** -8)
        else:
            close(tally.weights[r, :, : lengths[r]], want, off + want * 2.0 ** -23)


@pytest.mark.parametrize("heads,kv,dim", [(17, 1, 128), (18, 1, 128), (40, 2, 128), (23, 1, 128), (25, 1, 128), (48, 2, 128), (18, 1, 64), (48, 2, 64)])
def test_groups_of_more_heads_than_a_strip(heads, kv, dim):
    lengths = [1500, 0, 129, 64, 1, 700, 2900]
    cache, table, random = pages_of(lengths, kv, dim, 16, seed=heads)
    q, tally = queries(random, len(lengths), heads * dim), new_tally(len(lengths), kv, table.shape[1] * 16)
    out = attention_tallied(q, heads, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.zeros(len(lengths), dtype=torch.int32, device="cuda"), tally, dim ** -0.5)
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, [1] * len(lengths), lengths, dim ** -0.5):
        if e is not None:
            close(out[r], want, off + want.abs() * 2.0 ** -8)
        else:
            close(tally.weights[r, :, : lengths[r]], want, off + want * 2.0 ** -23)


@pytest.mark.parametrize("lengths", [[8192, 8001, 5], [4097]])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (32, 2, 64), (16, 1, 128)])
def test_requests_that_fill_a_cluster(heads, kv, dim, lengths):
    cache, table, random = pages_of(lengths, kv, dim, 64, seed=11, slack=0)
    q, tally = queries(random, len(lengths), heads * dim), new_tally(len(lengths), kv, 8192)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = attention_tallied(q, heads, cache, table, length, length, tally, dim ** -0.5)
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, [1] * len(lengths), lengths, dim ** -0.5):
        if e is not None:
            close(out[r], want, off + want.abs() * 2.0 ** -8)
        else:
            close(tally.weights[r, :, : lengths[r]], want, off + want * 2.0 ** -23)


def test_one_long_request():
    heads, kv, dim, page, lengths = 28, 4, 128, 64, [70001]
    cache, table, random = pages_of(lengths, kv, dim, page, seed=5)
    q, tally = queries(random, 1, heads * dim), new_tally(1, kv, 70016)
    out = attention_tallied(q, heads, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor([9], dtype=torch.int32, device="cuda"), tally, dim ** -0.5)
    ops.raise_on_status(q.device)
    (_, want, off, _), (_, weights, off_weights, _) = attended(q, heads, cache, table, [1], lengths, dim ** -0.5)
    close(out[0], want, off + want.abs() * 2.0 ** -8)
    close(tally.weights[0, :, :70001], weights, off_weights + weights * 2.0 ** -23)


def test_a_head_with_a_nan_or_an_infinity_is_nan_and_no_other_key_value_head_is():
    heads, kv, dim, page, lengths = 6, 3, 64, 16, [100, 100]
    cache, table, random = pages_of(lengths, kv, dim, page, seed=6)
    q, tally = queries(random, 2, heads * dim), new_tally(2, kv, 112)
    q[0, 2 * dim] = float("nan")               # head 2 of key/value head 1
    cache[table[1, 3], 0, 2, 5] = float("inf")  # a key of key/value head 2
    out = attention_tallied(q, heads, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor([99, 99], dtype=torch.int32, device="cuda"), tally, 0.125)
    ops.raise_on_status(q.device)
    bad = out.view(2, heads, dim).isnan().all(-1)
    assert bad.tolist() == [[False, False, True, False, False, False], [False] * 4 + [True, True]]
    assert out.isnan().view(2, heads, dim).any(-1).tolist() == bad.tolist()
    nan = tally.weights[:, :, :100].isnan()
    assert nan.all(-1).tolist() == nan.any(-1).tolist() == [[False, True, False], [False, False, True]]
    assert not tally.weights[:, :, 100:].isnan().any()


def test_scores_of_negative_infinity_give_nothing():
    """Keys of -infinity against positive queries: a slot that weighs nothing; where all are, the result is zeros."""
    lengths, dim, page = [40, 40], 64, 8
    cache, table, random = pages_of(lengths, 1, dim, page, seed=7)
    q = queries(random, 2, 2 * dim).abs() + 0.1
    cache[table[0, 1], 0] = float("-inf")
    cache[table[1, :5].long(), 0] = float("-inf")
    tally = new_tally(2, 1, 40)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = attention_tallied(q, 2, cache, table, length, length, tally, 0.125)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    assert bool((out[1] == 0).all()) and bool((tally.weights[1] == 0).all()) and bool((tally.weights[0, 0, 8:16] == 0).all()) and not out.isnan().any()
    assert abs(tally.weights[0].sum().item() - 2) < 1e-5
    tally_queries(q, 2, cache, table, starts, length, tally, 0.125, most=1)
    ops.raise_on_status(q.device)
    assert bool((tally.weights[1] == 0).all()) and abs(tally.weights[0].sum().item() - 4) < 1e-5


@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
@pytest.mark.parametrize("counts,lengths", [([1], [1]), ([5], [300]), ([1, 0, 33, 64], [64, 5, 33, 200]), ([130, 7], [130, 9]), ([32], [1500]), ([400, 150], [400, 900])])
def test_queries(heads, kv, dim, page, counts, lengths):
    if heads == 40 and sum(counts) > 300:
        counts = [n // 4 for n in counts]
    cache, table, random = pages_of(lengths, kv, dim, page, seed=sum(counts))
    q = queries(random, sum(counts) + 3, heads * dim, 16)  # rows behind the last request
    q[sum(counts):] = float("nan")
    tally = new_tally(len(counts), kv, table.shape[1] * page + 5)
    tally.weights.copy_(torch.rand(tally.weights.shape, generator=random))
    before, positions = tally.weights.clone(), tally.positions.clone()
    starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    tally_queries(q, heads, cache, table, starts, torch.tensor(lengths, dtype=torch.int32, device="cuda"), tally, dim ** -0.5, most=max(counts))
    ops.raise_on_status(q.device)
    assert torch.equal(positions, tally.positions)
    for r, want, off, e in attended(q, heads, cache, table, counts, lengths, dim ** -0.5):
        if e is None:
            n = lengths[r]
            want = want + before[r, :, :n].double()
            rows = counts[r] * heads // kv  # sums over the rows, a quarter of them by one lane one behind the other
            close(tally.weights[r, :, :n], want, off + want * (rows / 4 + 4) * 2.0 ** -24 + 2.0 ** -23)
            assert torch.equal(tally.weights[r, :, n:], before[r, :, n:])


@pytest.mark.parametrize("heads,kv,dim,page", [(14, 2, 64, 16), (28, 4, 128, 16), (16, 16, 64, 8), (32, 8, 128, 32), (24, 1, 128, 64)])
def test_a_few_queries_of_long_contexts(heads, kv, dim, page):
    """Rows of one tile, beside which tiles of slots pass; weights that slots have already are added to."""
    counts, lengths = [3, 0, 1, 5, 2, 4], [2900, 700, 1, 1537, 1, 128 * (9 if kv > 1 else 60)]
    counts[4] = 1
    cache, table, random = pages_of(lengths, kv, dim, page, seed=heads)
    q, tally = queries(random, sum(counts), heads * dim, 8), new_tally(len(lengths), kv, table.shape[1] * page)
    tally.weights.copy_(torch.rand(tally.weights.shape, generator=random))
    before = tally.weights.clone()
    starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    tally_queries(q, heads, cache, table, starts, torch.tensor(lengths, dtype=torch.int32, device="cuda"), tally, dim ** -0.5, most=max(counts))
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, counts, lengths, dim ** -0.5):
        if e is None:
            want = want + before[r, :, : lengths[r]].double()
            close(tally.weights[r, :, : lengths[r]], want, off + want * 2.0 ** -23)
            assert torch.equal(tally.weights[r, :, lengths[r]:], before[r, :, lengths[r]:])


def test_a_query_with_a_nan_spoils_the_slots_that_it_sees_and_no_others():
    cache, table, random = pages_of([300], 2, 64, 16, seed=12)
    q, tally = queries(random, 250, 6 * 64), new_tally(1, 2, 304)
    q[170, 64] = float("nan")   # a head of key/value head 0: sees slots 0 .. 220
    q[100, 5 * 64] = float("inf")  # of key/value head 1: slots 0 .. 150
    tally_queries(q, 6, cache, table, torch.tensor([0, 250], dtype=torch.int32, device="cuda"), torch.tensor([300], dtype=torch.int32, device="cuda"), tally, 0.125, most=250)
    ops.raise_on_status(q.device)
    assert [tally.weights[0, h].isnan().nonzero().flatten().tolist() for h in range(2)] == [list(range(221)), list(range(151))]


def test_prompts_of_many_spans():
    """Tiles of queries are cut into spans of 16, whose parts are put together."""
    counts, lengths, heads, kv, dim = [2500, 700], [2600, 3000], 8, 1, 64
    cache, table, random = pages_of(lengths, kv, dim, 64, seed=13)
    q, tally = queries(random, sum(counts), heads * dim, size=1.0), new_tally(2, kv, 3008)
    starts = torch.tensor([0, 2500, 3200], dtype=torch.int32, device="cuda")
    tally_queries(q, heads, cache, table, starts, torch.tensor(lengths, dtype=torch.int32, device="cuda"), tally, 0.125, most=2500)
    ops.raise_on_status(q.device)
    first = 0
    for r, (count, length) in enumerate(zip(counts, lengths)):
        k, _ = records(cache, table, r, length)
        y = torch.einsum("ihd,nd->ihn", q[first: first + count].double().view(count, heads, dim), k[0]) * 0.125
        y.masked_fill_((torch.arange(length, device="cuda") > torch.arange(length - count, length, device="cuda")[:, None])[:, None], float("-inf"))
        p = torch.softmax(y, -1)
        size = torch.einsum("ihd,nd->ihn", q[first: first + count].double().view(count, heads, dim).abs(), k[0].abs()).amax(-1, keepdim=True) * 0.125 * LOG2E
        e = 2 * (0.6931471805599453 * 2.0 ** -22 * ((dim / 16 + 4) * size + 20) + 2.0 ** -21) + 64 * 2.0 ** -24
        first += count
        close(tally.weights[r, 0, :length], p.sum((0, 1)), (p * e).sum((0, 1)) + p.sum((0, 1)) * 8 * 2.0 ** -24)


def test_more_queries_than_slots_see_nothing():
    cache, table, random = pages_of([3], 1, 64, 8, seed=2)
    q, tally = queries(random, 5, 2 * 64), new_tally(1, 1, 8)
    tally_queries(q, 2, cache, table, torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"), tally, 0.125, most=5)
    ops.raise_on_status(q.device)
    # queries 2, 3 and 4 see 1, 2 and 3 slots: two heads each
    assert abs(tally.weights.sum().item() - 6) < 1e-5 and bool((tally.weights[0, 0, 3:] == 0).all())


def test_a_prompt_and_its_tokens_one_by_one_leave_the_same_tally():
    """tally_queries over a prompt against attention_tallied token by token: each adds the same weights, in another order."""
    heads, kv, dim, page, n = 14, 2, 64, 16, 75
    cache, table, random = pages_of([n], kv, dim, page, seed=3)
    q, whole, step = queries(random, n, heads * dim), new_tally(1, kv, 96), new_tally(1, kv, 96)
    tally_queries(q, heads, cache, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda"), whole, 0.125, most=n)
    for i in range(n):
        at = torch.tensor([i + 1], dtype=torch.int32, device="cuda")
        attention_tallied(q[i: i + 1], heads, cache, table, at, at - 1, step, 0.125)
    ops.raise_on_status(q.device)
    assert torch.equal(whole.positions, step.positions)
    assert abs(whole.weights.sum().item() - heads * n) < 1e-3
    close(step.weights, whole.weights.double(), whole.weights.double() * 2.0 ** -14 + 1e-12)  # both off by e_p, some 2^-17 here


def test_pages_that_are_not_there_and_lengths_beyond_the_bound_are_reported():
    cache, table, random = pages_of([40], 1, 64, 8, seed=8)
    q, tally = queries(random, 1, 2 * 64), new_tally(1, 1, 48)
    one = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for call in (lambda t, n, longest: attention_tallied(q, 2, cache, t, one(n), one(0), tally, 0.125, longest=longest),
                 lambda t, n, longest: tally_queries(q, 2, cache, t, starts, one(n), tally, 0.125, most=1, longest=longest)):
        for page in (-1, cache.shape[0]):
            bad = table.clone()
            bad[0, 2] = page
            call(bad, 40, 40)
            with pytest.raises(ops.KernelError, match="block-table entry"):
                ops.raise_on_status(q.device)
        call(table, 41, 40)
        with pytest.raises(ops.KernelError, match="position"):
            ops.raise_on_status(q.device)
        call(table, 40, 40)
        ops.raise_on_status(q.device)
