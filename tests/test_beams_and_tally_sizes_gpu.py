"""Sizes at the ends: more requests than a warp's registers hold the tiles of, grids of many requests and groups, memory beyond 32 bits of bytes and of elements, bounds far above what is held.

Tolerances as in test_tally_gpu.py; what is moved is equal to the bit."""
from __future__ import annotations

import pytest
import torch
from test_beams_gpu import check_selection, some_logits
from test_tally_gpu import attended, close, pages_of, queries
from test_tally_queries_edges_gpu import ints

from hyperion_b200 import ops
from hyperion_b200.ops import Tally, attention_tallied, beam_reorder, evict, new_tally, tally_queries
from hyperion_b200.sampling import beam_select

pytestmark = pytest.mark.gpu


def check_token(lengths, heads, kv, dim, page=16, **bound):
    cache, table, random = pages_of(lengths, kv, dim, page, seed=len(lengths))
    q, tally = queries(random, len(lengths), heads * dim), new_tally(len(lengths), kv, table.shape[1] * page)
    out = attention_tallied(q, heads, cache, table, ints(lengths), ints(lengths), tally, dim ** -0.5, **bound)
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, [1] * len(lengths), lengths, dim ** -0.5):
        if e is not None:
            close(out[r], want, off + want.abs() * 2.0 ** -8)
        else:
            close(tally.weights[r, :, : lengths[r]], want, off + want * 2.0 ** -23)
            assert bool((tally.weights[r, :, lengths[r]:] == 0).all())


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (20, 1, 128), (40, 1, 64), (7, 1, 128)])
@pytest.mark.parametrize("requests", [127, 128, 129, 500])
def test_many_requests(requests, heads, kv, dim):
    check_token([(53 * i + i // 7) % 230 if i % 5 else 0 for i in range(requests)], heads, kv, dim)


@pytest.mark.parametrize("requests", [128, 700])
def test_many_requests_of_nothing(requests):
    check_token([0] * requests, 8, 4, 64)
    check_token([0] * (requests - 1) + [70], 8, 4, 64)
    check_token([1] + [0] * (requests - 1), 8, 4, 64)


def test_the_most_requests():
    """As many as a grid has; one more is refused.  S is below 14 here, e_p then below 2^-14, and a result, of values below 6, off by less than 2^-12 beside its rounding."""
    requests, dim, random = 65535, 64, torch.Generator("cuda").manual_seed(9)
    cache = torch.randn(8, 2, 1, 8, dim, device="cuda", generator=random).to(torch.bfloat16)
    table = (torch.arange(requests, device="cuda") % 8).to(torch.int32)[:, None].contiguous()
    q = torch.randn(requests + 1, dim, device="cuda", generator=random).to(torch.bfloat16)
    lengths, tally = torch.full((requests,), 3, dtype=torch.int32, device="cuda"), new_tally(requests, 1, 8)
    out = attention_tallied(q[:requests], 1, cache, table, lengths, lengths, tally, 0.125)
    keys, values = cache[table[:, 0].long(), 0, 0, :3].double(), cache[table[:, 0].long(), 1, 0, :3].double()
    p = torch.softmax(torch.einsum("rd,rnd->rn", q[:requests].double(), keys) * 0.125, -1)
    assert bool(((tally.weights[:, 0, :3] - p).abs() <= p * 2.0 ** -14 + 2.0 ** -24).all())
    want = torch.einsum("rn,rnd->rd", p, values)
    assert values.abs().max().item() < 6 and torch.einsum("rd,rnd->rn", q[:requests].abs().double(), keys.abs()).max().item() * 0.125 * 1.4427 < 14
    assert bool(((out - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -12).all())
    tally_queries(q[:requests], 1, cache, table, torch.arange(requests + 1, dtype=torch.int32, device="cuda"), lengths, tally, 0.125, most=1)
    assert bool(((tally.weights[:, 0, :3] - 2 * p).abs() <= p * 2.0 ** -13 + 2.0 ** -23).all())
    left = evict(cache, table, lengths, lengths - 1, tally, 3)
    assert bool((left == 3).all())
    ops.raise_on_status(q.device)
    more = torch.zeros(requests + 1, 1, dtype=torch.int32, device="cuda")
    for call in (lambda: attention_tallied(q, 1, cache, more, more[:, 0].contiguous(), more[:, 0].contiguous(), new_tally(requests + 1, 1, 8), 0.125),
                 lambda: tally_queries(q, 1, cache, more, torch.zeros(requests + 2, dtype=torch.int32, device="cuda"), more[:, 0].contiguous(), new_tally(requests + 1, 1, 8), 0.125, most=1),
                 lambda: evict(cache, more, more[:, 0].contiguous(), more[:, 0].contiguous(), new_tally(requests + 1, 1, 8), 3)):
        with pytest.raises(ops.KernelError, match="unsupported size"):
            call()


def test_many_requests_queries():
    heads, kv, dim, page, requests = 6, 2, 64, 8, 300
    counts = [i % 4 for i in range(requests)]
    lengths = [max(n, (31 * i) % 200) for i, n in enumerate(counts)]
    cache, table, random = pages_of(lengths, kv, dim, page, seed=3)
    q, tally = queries(random, sum(counts), heads * dim), new_tally(requests, kv, table.shape[1] * page)
    starts = [sum(counts[:i]) for i in range(requests + 1)]
    tally_queries(q, heads, cache, table, ints(starts), ints(lengths), tally, 0.125, most=3)
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, counts, lengths, 0.125):
        if e is None:
            close(tally.weights[r, :, : lengths[r]], want, off + want * 16 * 2.0 ** -24)


def moved_far(pages, kv, page, dim, table, random):
    """A cache of more than 2^32 bytes of which only the table's pages hold anything, and a small one that holds the same."""
    cache = torch.empty(pages, 2, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    near = torch.randn(table.numel(), 2, kv, page, dim, generator=random).to(torch.bfloat16).cuda()
    cache[table.flatten().long()] = near
    return cache, near, torch.arange(table.numel(), dtype=torch.int32, device="cuda").view(table.shape)


def test_pages_beyond_32_bits():
    kv, page, dim, heads, pages = 4, 64, 128, 28, 40000  # 131,072 bytes a page: 5.2 GB; rows of 128 up to 2^24
    random = torch.Generator().manual_seed(1)
    table = torch.tensor([[39999, 3, 32768], [32767, 39998, 16384], [20000, 16383, 35000]], dtype=torch.int32).cuda()
    cache, near, near_table = moved_far(pages, kv, page, dim, table, random)
    q, many, lengths = queries(random, 3, heads * dim), queries(random, 60, heads * dim), ints([192, 130, 7])
    found = []
    for pool, blocks in ((cache, table), (near, near_table)):
        tally = new_tally(3, kv, 192)
        out = attention_tallied(q, heads, pool, blocks, lengths, lengths, tally, dim ** -0.5)
        tally_queries(many, heads, pool, blocks, ints([0, 50, 53, 60]), lengths, tally, dim ** -0.5, most=50)
        left = evict(pool, blocks, lengths, lengths - 1, tally, 60, first=1, recent=3)
        beam_blocks = blocks.clone()
        beam_reorder(ints([[2, 0, 1]]), ints([50]), beam_blocks, [pool.view(1, -1, 2 * kv, page, dim)], [tally.weights.view(1, 3, -1)])
        found.append([out.view(torch.int16), tally.weights, tally.positions, left, pool[blocks.flatten().long()].view(torch.int16)])
    ops.raise_on_status(q.device)
    assert all(torch.equal(a, b) for a, b in zip(*found))


def test_layers_beyond_32_bits():
    """Eviction and reordering over layers, 2.1e9 entries and more apart."""
    layers, kv, page, dim, pages = 3, 2, 16, 64, 700000  # 8,192 bytes a page: 5.7 GB a layer
    random = torch.Generator().manual_seed(2)
    table = torch.tensor([[699999, 1, 524288, 300000]], dtype=torch.int32).cuda()
    cache = torch.empty(layers, pages, 2, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    near = torch.randn(layers, 4, 2, kv, page, dim, generator=random).to(torch.bfloat16).cuda()
    cache[:, table[0].long()] = near
    weights, lengths, found = torch.rand(layers, 1, kv, 64, generator=random).cuda(), ints([61]), []
    for pool, blocks in ((cache, table), (near, ints([[0, 1, 2, 3]]))):
        tally = Tally(weights.clone(), torch.arange(64, dtype=torch.int32, device="cuda").expand(weights.shape).contiguous())
        left = evict(pool, blocks, lengths, lengths - 1, tally, 23, first=1, recent=4)
        two = blocks.view(2, 2).clone()
        beam_reorder(ints([[1, 0]]), ints([21]), two, [pool.view(layers, -1, 2 * kv, page, dim)])
        found.append([left, *tally, pool[:, blocks[0].long()].view(torch.int16)])
    ops.raise_on_status(lengths.device)
    assert all(torch.equal(a, b) for a, b in zip(*found))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_logits_beyond_32_bits(dtype):
    logits, scores = some_logits(2, 5, 20000, dtype, seed=4)
    stride = (1 << 29) + 24
    far = torch.empty(9 * stride + 20000, dtype=dtype, device="cuda").as_strided((10, 20000), (stride, 1))
    far.copy_(logits)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(far, scores, 10), beam_select(logits, scores, 10)))


def test_the_most_rows_of_logits():
    logits, _ = some_logits(65535, 1, 40, seed=6)
    choice = beam_select(logits, torch.zeros(65535, 1, device="cuda"), 2)
    want = logits.sort(dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(choice.tokens.long(), want) and bool((choice.parents == 0).all())
    with pytest.raises(ops.KernelError, match="unsupported size"):
        beam_select(torch.zeros(65536, 4, device="cuda"), torch.zeros(65536, 1, device="cuda"), 2)
    check_selection(*some_logits(700, 3, 77, seed=7), 5)


def test_many_groups_of_beams():
    groups, beams = 3000, 4
    state = torch.randn(2, groups * beams, 5, device="cuda")
    parents = torch.randint(0, beams, (groups, beams), dtype=torch.int32, device="cuda")
    want = state.view(2, groups, beams, 5).gather(2, parents.long()[None, :, :, None].expand(2, -1, -1, 5)).view(state.shape)
    beam_reorder(parents, torch.zeros(groups, dtype=torch.int32, device="cuda"), None, [], [state])
    ops.raise_on_status(state.device)
    assert torch.equal(state, want)


def test_a_bound_far_above_what_is_held():
    """Rows of scores more than 2^31 entries behind the first."""
    heads, kv, dim, page, lengths = 64, 8, 64, 64, [100, 1, 0, 640, 64, 65, 300, 7]
    cache, table, random = pages_of(lengths, kv, dim, page, seed=8)
    bound = 4_400_000
    wide = torch.full((len(lengths), bound // page + 1), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    q, tally = queries(random, len(lengths), heads * dim), new_tally(len(lengths), kv, bound)
    out = attention_tallied(q, heads, cache, wide, ints(lengths), ints(lengths), tally, dim ** -0.5, longest=bound)
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(q, heads, cache, table, [1] * len(lengths), lengths, dim ** -0.5):
        if e is not None:
            close(out[r], want, off + want.abs() * 2.0 ** -8)
        else:
            close(tally.weights[r, :, : lengths[r]], want, off + want * 2.0 ** -23)
    again = new_tally(len(lengths), kv, bound)
    counts = [min(n, 3) for n in lengths]
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    many = queries(random, sum(counts), heads * dim)
    tally_queries(many, heads, cache, wide, ints(starts), ints(lengths), again, dim ** -0.5, most=3, longest=bound)
    ops.raise_on_status(q.device)
    for r, want, off, e in attended(many, heads, cache, table, counts, lengths, dim ** -0.5):
        if e is None:
            close(again.weights[r, :, : lengths[r]], want, off + want * 16 * 2.0 ** -24)
