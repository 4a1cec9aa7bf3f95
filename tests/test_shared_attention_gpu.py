"""Attention behind shared positions against plain attention in 64 bits over the same records.

Tolerance: weights are rounded once (bfloat16, 2^-9, over bfloat16 caches; float16, 2^-12, over 8-bit ones) and so is the result (2^-9); what float32 adds (scores of up
to some 50 in the exponent, sums of up to 10^4 weights) is below 2^-12.  An entry is off by at most (2^-8 + 2^-11) * sum_j p_j |v_j|."""
from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops.cache8 import Cache8
from hyperion_b200.ops.shared import attention_shared, plan_shared

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def records(random, pages, kv, page, dim, bits):
    x = torch.randn(pages, 2, kv, page, dim, device="cuda", generator=random)
    if bits == 16:
        return x.to(BF)
    exponents = torch.randint(-9, -5, (pages, 2, kv, page), device="cuda", generator=random)
    return Cache8((x * 128).clamp(-448, 448).to(torch.float8_e4m3fn), exponents.to(torch.int8))


def values(cache):
    if isinstance(cache, Cache8):
        return cache.codes.double() * torch.exp2(cache.exponents.double())[..., None]
    return cache.double()


def step(counts, lengths, heads, kv, dim, page, bits, groups=(), seed=0, spare=2):
    """Queries, a cache and block tables in which the requests of a group hold the same pages for the positions they share."""
    random = torch.Generator("cuda").manual_seed(seed)
    blocks = max(1, -(-max(lengths) // page))
    table = torch.randperm(len(counts) * blocks + spare, device="cuda", generator=random)[: len(counts) * blocks].to(torch.int32).view(len(counts), blocks)
    cache = records(random, len(counts) * blocks + spare, kv, page, dim, bits)
    for first, n, positions in groups:
        whole = positions // page
        table[first: first + n, :whole] = table[first, :whole].clone()
        for i in range(first, first + n):  # the page that the shared positions end in is each request's own copy
            if positions % page:
                for part in (cache if isinstance(cache, Cache8) else (cache,)):
                    part.view(torch.uint8 if bits == 8 else part.dtype)[int(table[i, whole]), :, :, : positions % page] = \
                        part.view(torch.uint8 if bits == 8 else part.dtype)[int(table[first, whole]), :, :, : positions % page].clone()
    q = torch.randn(sum(counts), heads * dim, device="cuda", generator=random).to(BF)
    return q, cache, table


def plain(q, heads, cache, table, counts, lengths, scale):
    """(result, sum of p |v|) [tokens, heads * dim] in 64 bits; only the positions that a request holds are looked at."""
    dense = values(cache)
    kv, page, dim = dense.shape[2:]
    out, size, first = [], [], 0
    for r, (n, length) in enumerate(zip(counts, lengths)):
        k, v = dense[table[r, : -(-length // page)].long()].permute(1, 2, 0, 3, 4).reshape(2, kv, -1, dim)[:, :, :length].repeat_interleave(heads // kv, 1)
        for i in range(n):
            x = q[first + i, : heads * dim].double().view(heads, 1, dim)
            seen = max(0, length - n + i + 1)
            p = torch.softmax(x @ k[:, :seen].transpose(1, 2) * scale, -1) if seen else x.new_zeros(heads, 1, 0)
            out.append((p @ v[:, :seen]).reshape(-1))
            size.append((p @ v[:, :seen].abs()).reshape(-1))
        first += n
    return torch.stack(out), torch.stack(size)


def agree(got, want, size):
    ops.raise_on_status(got.device)
    assert got.dtype == BF
    assert ((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * size + 1e-30).all(), float(((got.double() - want).abs() / (size + 1e-30)).max())


def check(counts, lengths, heads, kv, dim, page, bits, groups=(), seed=0, scale=None):
    q, cache, table = step(counts, lengths, heads, kv, dim, page, bits, groups, seed)
    scale = scale or dim ** -0.5
    plan = plan_shared(counts, lengths, heads, kv, dim, shared=groups)
    got = attention_shared(q, heads, cache, table, plan, scale)
    agree(got, *plain(q, heads, cache, table, counts, lengths, scale))
    assert torch.equal(got, attention_shared(q, heads, cache, table, plan, scale))  # the order of the sums is fixed
    return got


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (28, 4, 128), (4, 4, 128), (8, 1, 64), (40, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("page", [8, 64])
def test_head_layouts(heads, kv, dim, page, bits):
    check([1, 3, 1], [200, 77, 1], heads, kv, dim, page, bits)
    check([1, 2, 1, 1], [300, 290, 257, 258], heads, kv, dim, page, bits, groups=[(0, 4, 256)], seed=1)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 191, 1000, 5000])
def test_lengths(length, bits):
    check([1], [length], 8, 2, 128, 16, bits)
    check([1, 1, 1], [length + 1, length + 70, length + 1], 8, 2, 64, 32, bits, groups=[(0, 3, length)])


@pytest.mark.parametrize("bits", [8, 16])
def test_groups_of_every_kind(bits):
    """Requests of no group before, between and after groups; groups of one; a group whose first request is not in the step; queries in number."""
    counts, lengths = [2, 1, 5, 1, 0, 1, 3, 1, 1, 4], [90, 150, 160, 140, 130, 131, 333, 70, 64, 4]
    check(counts, lengths, 12, 4, 128, 16, bits, groups=[(1, 3, 139), (4, 2, 100), (6, 1, 64), (7, 2, 0)])


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("counts,lengths", [([200], [200]), ([33, 65], [33, 700]), ([300], [1301]), ([40, 1, 90], [41, 2000, 90])])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (8, 8, 128), (16, 4, 128)])
def test_portions_of_prompts(counts, lengths, heads, kv, dim, bits):
    check(counts, lengths, heads, kv, dim, 16, bits)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("requests,shared", [(70, 513), (150, 1000), (40, 3001)])
def test_many_requests_behind_one_prefix(requests, shared, bits):
    random = np.random.default_rng(requests)
    counts = random.integers(1, 4, requests).tolist()
    lengths = [shared + c + int(x) for c, x in zip(counts, random.integers(0, 200, requests))]
    check(counts, lengths, 14, 2, 64, 16, bits, groups=[(0, requests, shared)])
    check(counts, lengths, 8, 2, 128, 64, bits, groups=[(0, requests // 2, shared), (requests // 2, requests - requests // 2, shared - 100)])


@pytest.mark.parametrize("bits", [8, 16])
def test_rows_that_see_nothing(bits):
    got = check([3, 1, 2], [1, 0, 500], 8, 2, 128, 16, bits)
    assert (got[:2] == 0).all() and (got[3] == 0).all() and (got[2] != 0).any()
    assert (check([1, 2], [0, 0], 8, 2, 64, 16, bits) == 0).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("groups", [(), ((0, 3, 100),)])
def test_what_lies_beyond_a_length_does_not_matter(bits, groups):
    counts, lengths = [1, 2, 40], [101, 130, 333]
    q, cache, table = step(counts, lengths, 8, 2, 128, 16, bits, groups)
    plan = plan_shared(counts, lengths, 8, 2, 128, shared=groups)
    want = attention_shared(q, 8, cache, table, plan, 0.1)
    unused = torch.ones(cache[0].shape[0] if bits == 8 else cache.shape[0], 16, dtype=torch.bool, device="cuda")
    for r, length in enumerate(lengths):
        for p in range(length):
            unused[int(table[r, p // 16]), p % 16] = False
    at = unused.nonzero(as_tuple=True)
    for bad in (float("nan"), float("inf"), -3e38):
        if bits == 8:
            cache.codes.view(torch.uint8)[at[0], :, :, at[1]] = 0x7F if bad != bad else 0xFE
            cache.exponents[at[0], :, :, at[1]] = 127 if bad == float("inf") else -128
        else:
            cache[at[0], :, :, at[1]] = bad
        assert torch.equal(want, attention_shared(q, 8, cache, table, plan, 0.1)), bad


def test_a_nan_in_a_seen_place_stays_one():
    q, cache, table = step([1, 1], [70, 70], 2, 1, 64, 16, 8)
    cache.codes.view(torch.uint8)[int(table[0, 2]), 1, 0, 3, 5] = 0x7F
    got = attention_shared(q, 2, cache, table, plan_shared([1, 1], [70, 70], 2, 1, 64), 0.1)
    assert torch.isnan(got[0].view(2, 64)[:, 5]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("counts,lengths,groups", [([3], [200], ()), ([300], [1301], ()), ([1] * 70, [700] * 70, ((0, 70, 513),))])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("bits", [8, 16])
def test_rows_that_see_a_key_without_a_number(bits, bad, counts, lengths, groups):
    """A NaN or a positive infinity among a row's scores makes the row NaN; a negative infinity is a weight of 0; rows that do not see the key stay as they are."""
    if bits == 8 and bad == "inf":
        return  # e4m3 has no infinity
    q, cache, table = step(counts, lengths, 8, 2, 128, 16, bits, groups, seed=8)
    at = lengths[0] - counts[0] + counts[0] // 2 if not groups else 300
    place = int(table[0, at // 16]), 0, 1, at % 16, 7  # an entry of a key of the second key/value head
    if bits == 8:
        cache.codes.view(torch.uint8)[place] = 0x7F
    else:
        cache[place] = float(bad)
    got = attention_shared(q, 8, cache, table, plan_shared(counts, lengths, 8, 2, 128, shared=groups), 0.1)
    ops.raise_on_status(got.device)
    want, size = plain(q, 8, cache, table, counts, lengths, 0.1)
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    agree(torch.nan_to_num(got), torch.nan_to_num(want), torch.nan_to_num(size))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_large_and_small_scores(bits, size):
    """Nearly equal weights, and one key that takes all; queries near bfloat16's ends keep their digits (the scale brings the scores back)."""
    for q_size in (1.0, 1e30, 1e-30):
        q, cache, table = step([1, 2, 50], [900, 500, 300], 8, 2, 128, 16, bits, seed=5)
        q = (q.float() * q_size).to(BF)
        scale = size / q_size / 128 ** 0.5
        got = attention_shared(q, 8, cache, table, plan_shared([1, 2, 50], [900, 500, 300], 8, 2, 128), scale)
        agree(got, *plain(q, 8, cache, table, [1, 2, 50], [900, 500, 300], scale))


def test_exponents_far_apart():
    """Values of very different sizes in one row: the small ones' weights still count in the sum."""
    q, cache, table = step([1, 30], [300, 300], 4, 1, 128, 16, 8, seed=6)
    random = torch.Generator("cuda").manual_seed(7)
    cache.exponents[:, 1] = torch.randint(-40, 41, cache.exponents[:, 1].shape, device="cuda", generator=random).to(torch.int8)
    cache.exponents[:, 0] = torch.randint(-14, -6, cache.exponents[:, 0].shape, device="cuda", generator=random).to(torch.int8)
    got = attention_shared(q, 4, cache, table, plan_shared([1, 30], [300, 300], 4, 1, 128), 0.1)
    agree(got, *plain(q, 4, cache, table, [1, 30], [300, 300], 0.1))
    cache.exponents[:, 1] = -40
    cache.exponents[int(table[0, 3]), 1, :, 5] = 40
    cache.codes.view(torch.uint8)[int(table[0, 3]), 1, :, 5] = 0
    got = attention_shared(q, 4, cache, table, plan_shared([1, 30], [300, 300], 4, 1, 128), 0.1)
    agree(got, *plain(q, 4, cache, table, [1, 30], [300, 300], 0.1))


@pytest.mark.parametrize("bits", [8, 16])
def test_strides_and_streams(bits):
    counts, lengths, groups = [1, 4, 60], [130, 140, 300], [(0, 2, 120)]
    q, cache, table = step(counts, lengths, 8, 2, 64, 16, bits, groups)
    plan = plan_shared(counts, lengths, 8, 2, 64, shared=groups)
    want = attention_shared(q, 8, cache, table, plan, 0.125)
    wide = torch.randn(q.shape[0], 3 * 8 * 64 + 8, device="cuda").to(BF)
    wide[:, 512:1024] = q
    out = torch.full((q.shape[0], 700), 3.0, device="cuda", dtype=BF)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = attention_shared(wide[:, 512:], 8, cache, table, plan, 0.125, out=out)
    stream.synchronize()
    assert torch.equal(got[:, :512], want) and (out[:, 512:] == 3).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (28, 4, 128), (40, 2, 128)])
@pytest.mark.parametrize("counts,lengths", [([1] * 5, [1500, 0, 1, 130, 800]), ([1] * 5, [1500, 3, 1, 130, 800]), ([2, 1, 2], [700, 1100, 2]), ([1], [640]), ([1] * 30, list(range(500, 1100, 20)))])
def test_runs_of_a_cluster(heads, kv, dim, counts, lengths, bits):
    """Runs whose shares are joined by the blocks themselves: of few blocks and of eight, some without a key.  (A row that sees nothing is left to the kernel behind.)"""
    assert (plan_shared(counts, lengths, heads, kv, dim).together > 0) == (0 not in lengths)
    check(counts, lengths, heads, kv, dim, 16, bits, seed=11)


def test_threads_on_one_stream():
    """Calls of several kernels from threads that launch on the same stream do not write over one another's pieces."""
    def work(seed):
        counts, lengths = [1] * 8, [2000 + 37 * seed + r for r in range(8)]
        q, cache, table = step(counts, lengths, 14, 2, 64, 16, 8, seed=seed)
        plan = plan_shared(counts, lengths, 14, 2, 64)
        assert plan.joined
        want = attention_shared(q, 14, cache, table, plan, 0.1)
        return all(torch.equal(want, attention_shared(q, 14, cache, table, plan, 0.1)) for _ in range(300))

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))


def test_pages_behind_32_bit_offsets():
    pages = 2**32 // (2 * 8 * 64 * 128) + 30
    random = torch.Generator("cuda").manual_seed(8)
    codes = torch.empty((pages, 2, 8, 64, 128), dtype=torch.uint8, device="cuda")
    exponents = torch.full((pages, 2, 8, 64), -8, dtype=torch.int8, device="cuda")
    table = torch.tensor([[pages - 1, 3, pages - 7, pages // 2 + 1], [pages - 2, pages - 3, 0, 1]], dtype=torch.int32, device="cuda")
    for p in table.view(-1).tolist():
        codes[p] = (torch.randn(2, 8, 64, 128, device="cuda", generator=random) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    cache = Cache8(codes.view(torch.float8_e4m3fn), exponents)
    q = torch.randn(71, 16 * 128, device="cuda", generator=random).to(BF)
    got = attention_shared(q, 16, cache, table, plan_shared([1, 70], [250, 240], 16, 8, 128), 0.09)
    used, small = table.view(-1).long(), torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    of_used = Cache8(codes[used].view(torch.float8_e4m3fn), exponents[used])
    agree(got, *plain(q, 16, of_used, small, [1, 70], [250, 240], 0.09))


def test_a_missing_page_is_reported():
    q, cache, table = step([1, 1], [100, 100], 2, 1, 64, 16, 8)
    table[1, 3] = cache.codes.shape[0]
    attention_shared(q, 2, cache, table, plan_shared([1, 1], [100, 100], 2, 1, 64), 0.1)
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.raise_on_status(q.device)


def test_refusals():
    q, cache, table = step([1, 1], [100, 100], 4, 2, 64, 16, 8)
    plan = plan_shared([1, 1], [100, 100], 4, 2, 64)
    good = dict(q=q, heads=4, cache=cache, block_table=table, plan=plan, scale=0.1)
    wide = records(torch.Generator("cuda").manual_seed(0), 20, 2, 16, 96, 16)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[:, :200]), dict(heads=2), dict(cache=cache.codes), dict(cache=wide), dict(block_table=table.long()), dict(block_table=table[:1]),
                dict(block_table=table[:, :6].contiguous()), dict(block_table=table.t().contiguous().t()), dict(cache=cache._replace(exponents=cache.exponents[1:])), dict(q=q.cpu()),
                dict(out=torch.empty(2, 256, device="cuda")), dict(q=torch.zeros(2, 260, device="cuda", dtype=BF)[:, 1:257])):
        with pytest.raises(ops.KernelError):
            attention_shared(**{**good, **bad})
    assert attention_shared(q[:0], 4, cache, table, plan_shared([0, 0], [100, 100], 4, 2, 64), 0.1).shape == (0, 256)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (16, 4, 128)])
def test_blocks_of_several_items(heads, kv, dim, bits):
    """More items than the device has multiprocessors, of many key tiles and of both heights, one behind the other in a block."""
    counts, lengths = [1500, 9, 70, 260], [5000, 300, 3000, 2000]
    q, cache, table = step(counts, lengths, heads, kv, dim, 16, bits, seed=9)
    plan = plan_shared(counts, lengths, heads, kv, dim)
    got = attention_shared(q, heads, cache, table, plan, 0.1)
    ops.raise_on_status(q.device)
    dense, first = values(cache), 0
    for r, (n, length) in enumerate(zip(counts, lengths)):
        k, v = dense[table[r, : -(-length // 16)].long()].permute(1, 2, 0, 3, 4).reshape(2, kv, 1, -1, dim)[:, :, :, :length]
        x = q[first: first + n].double().view(n, kv, heads // kv, dim).permute(1, 2, 0, 3)
        hidden = torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda")[:, None]
        p = torch.softmax((x @ k.transpose(2, 3) * 0.1).masked_fill(hidden, -float("inf")), -1)
        want, size = ((p @ y).permute(2, 0, 1, 3).reshape(n, -1) for y in (v, v.abs()))
        agree(got[first: first + n], want, size)
        first += n
