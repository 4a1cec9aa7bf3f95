"""Attention of a step over paged caches (bfloat16, or 8-bit records: :mod:`.cache8`) in which groups of requests share their first positions.

The requests of a group hold the same pages for their first positions (a system prompt, a document, the prompt that several drafts continue).
Token by token those pages would be fetched once per request; here a group's tokens walk them together, each request walks what it holds beyond
them, and the pieces of a row are put together (csrc/attention_shared.cu).  Requests that share nothing are groups of their own.

A step is planned on the host from its lengths (:func:`plan_shared`); every layer of the step runs from that plan (:func:`attention_shared`).
"""
from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

from . import native
from .basic import status_word
from .cache8 import Cache8, check_cache8
from .native import KernelError, check, f32, library, ptr, require_cuda, sm_count, stream_ptr

STRIP_ROWS = 8, 16  # (token, head) rows of a strip: eight where no request has more
TILE_ROWS = 256    # of an item of the tile kernel
STRIP_KEYS, TILE_KEYS = 128, 128  # keys that shares are counted in
STRIPS_PER_SM = {8: 3, 16: 2}  # blocks of the strip kernel that share an SM
# What an item costs beside its key tiles, in key tiles (its queries' way in, its rows' way out, the first tile's latency), and the least it is cut to.
STRIP_OVERHEAD, LEAST_STRIP = 3, 2
TILE_OVERHEAD, LEAST_TILES = 3, 2
MOST_STRIP_ROWS = 64
ITEM_WORDS = 6


def supported(head_dim: int, page_size: int) -> bool:
    return head_dim in (64, 128) and page_size in (8, 16, 32, 64)


class SharedPlan:
    """What the launches of a step need: the items, the last position each token sees and the first piece of each token, in one int32 tensor."""

    __slots__ = ("tokens", "rows", "heads", "kv_heads", "head_dim", "longest", "pieces", "joined", "strips", "strip_rows", "tiles", "data", "strips_at", "tiles_at", "last_at", "starts_at")


def _tiles_of(first, last, keys):
    return -(-last // keys) - first // keys


def _share(tiles, cuts, across, slots, overhead, least) -> int:
    """Key tiles of an item's share: the longest that lets the items take the device's ``slots`` in one to four turns, whichever is soonest done.
    An item costs ``overhead`` key tiles beside its own."""
    best = None
    for turns in range(1, 5):
        low, high = least, max(least, int(tiles.max()))  # the smallest share with no more items than that
        while low < high:
            middle = (low + high) // 2
            if int((cuts * -(-tiles // middle)).sum()) * across <= turns * slots:
                high = middle
            else:
                low = middle + 1
        items = int((cuts * -(-tiles // low)).sum()) * across
        time = -(-items // slots) * (low + overhead)
        if best is None or time < best[0]:
            best = time, low
    return best[1]


def _cut(first, last, keys, share):
    """Ranges [first, last) cut on tile boundaries into shares of about ``share`` tiles of ``keys``: (shares of each, source range, share's number, first key, last key + 1)."""
    base, tiles = first // keys, _tiles_of(first, last, keys)
    shares = np.maximum(1, -(-tiles // share))
    each = -(-tiles // shares)
    shares = -(-tiles // each)  # no share is empty
    source = np.repeat(np.arange(len(first)), shares)
    number = np.arange(len(source)) - np.repeat(np.cumsum(shares) - shares, shares)
    low = np.maximum(first[source], (base[source] + number * each[source]) * keys)
    high = np.minimum(last[source], (base[source] + (number + 1) * each[source]) * keys)
    return shares, source, number, low, high


def plan_shared(counts: Sequence[int], lengths: Sequence[int], heads: int, kv_heads: int, head_dim: int, *, shared: Sequence[tuple[int, int, int]] = (),
                device="cuda", sms: int | None = None) -> SharedPlan:
    """Plan a step of ``counts[r]`` queries of request r, whose block table (row r) holds ``lengths[r]`` positions: token i of n sees the first
    ``lengths[r] - n + i + 1`` of them (one with nothing to see comes out as zeros).  ``shared``: (first request, requests, positions) of each group
    of consecutive requests that hold the same pages for their first positions, which all of their queries see; in order, none of them overlapping."""
    n = np.asarray(counts, dtype=np.int64)
    length = np.asarray(lengths, dtype=np.int64)
    if n.ndim != 1 or n.shape != length.shape or (n < 0).any() or (length < 0).any():
        raise KernelError("plan_shared: a count of queries and a length for each request, none of them negative")
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise KernelError(f"plan_shared: {heads} query heads do not divide over {kv_heads} key/value heads")
    requests, total = len(n), int(n.sum())
    if length.size and int(length.max()) > 2**31 - 1 - TILE_KEYS:
        raise KernelError("plan_shared: a position fits 32 bits")
    start = np.concatenate([[0], np.cumsum(n)])
    own_from = np.zeros(requests, dtype=np.int64)
    groups, after = [], 0
    for first, members, positions in shared:
        if first < after or members < 0 or first + members > requests or positions < 0:
            raise KernelError("plan_shared: groups of consecutive requests, in order, that do not overlap")
        after = first + members
        inside = slice(first, after)
        if positions and ((length[inside] - n[inside] < positions) & (n[inside] > 0)).any():
            raise KernelError(f"plan_shared: every query of a group sees all of its {positions} shared positions")
        if positions and start[after] > start[first]:
            own_from[inside] = positions
            table_row = first + int(np.flatnonzero(n[inside])[0])  # of a request that is in the step
            groups.append((start[first], start[after] - start[first], table_row, positions, first, members))
    group_ranges = np.array(groups, dtype=np.int64).reshape(-1, 6)
    live = np.flatnonzero((n > 0) & (length > own_from))
    # ranges: (first token, tokens, table row, first key, last key + 1)
    ranges = np.concatenate([np.stack([group_ranges[:, 0], group_ranges[:, 1], group_ranges[:, 2], 0 * group_ranges[:, 3], group_ranges[:, 3]], 1),
                             np.stack([start[live], n[live], live, own_from[live], length[live]], 1)])
    group, sms = heads // kv_heads, sms or sm_count(device)
    shares, kinds = np.ones(len(ranges), dtype=np.int64), []
    wide = ranges[:, 1] * group > MOST_STRIP_ROWS
    strip_rows = STRIP_ROWS[int((ranges[~wide, 1] * group > STRIP_ROWS[0]).any())]
    for chosen, rows, keys, slots, overhead, least in ((np.flatnonzero(~wide), strip_rows, STRIP_KEYS, STRIPS_PER_SM[strip_rows] * sms, STRIP_OVERHEAD, LEAST_STRIP),
                                                       (np.flatnonzero(wide), TILE_ROWS, TILE_KEYS, sms, TILE_OVERHEAD, LEAST_TILES)):
        of_kind, per = ranges[chosen], max(1, rows // group)  # tokens of an item
        cuts = -(-of_kind[:, 1] // per)
        if len(chosen):
            parts, source, number, low, high = _cut(of_kind[:, 3], of_kind[:, 4], keys,
                                                     _share(_tiles_of(of_kind[:, 3], of_kind[:, 4], keys), cuts, kv_heads * -(-group // rows), slots, overhead, least))
            shares[chosen] = parts
            kinds.append((of_kind, chosen, per, cuts, source, number, low, high))
        else:
            kinds.append(None)
    # a token's pieces: its group's shares, then its own request's
    of_group = np.zeros(requests, dtype=np.int64)
    for k, (*_, first, members) in enumerate(groups):
        of_group[first: first + members] = shares[k]
    of_own = np.zeros(requests, dtype=np.int64)
    of_own[live] = shares[len(groups):]
    before = np.concatenate([np.zeros(len(groups), dtype=np.int64), of_group[live]])
    token_pieces = np.repeat(of_group + of_own, n)
    starts = np.concatenate([[0], np.cumsum(token_pieces)])
    # items: every share of a range for every run of `per` tokens of it, the longest first
    items = []
    for kind in kinds:
        if kind is None:
            items.append(np.zeros((0, ITEM_WORDS), dtype=np.int64))
            continue
        of_kind, chosen, per, cuts, source, number, low, high = kind
        times = cuts[source]
        at = np.repeat(np.arange(len(source)), times)
        run = np.arange(len(at)) - np.repeat(np.cumsum(times) - times, times)
        of = of_kind[source[at]]
        tok = of[:, 0] + run * per
        made = np.stack([tok, np.minimum(per, of[:, 0] + of[:, 1] - tok), of[:, 2], low[at], high[at], (number + before[chosen][source])[at]], 1)
        items.append(made[np.argsort(made[:, 3] - made[:, 4], kind="stable")])
    last = np.arange(total) - np.repeat(start[:-1], n) + np.repeat(length - n, n)

    plan = SharedPlan()
    plan.tokens, plan.rows, plan.heads, plan.kv_heads, plan.head_dim = total, requests, heads, kv_heads, head_dim
    plan.longest = int(length[n > 0].max()) if total else 0
    plan.pieces, plan.joined = int(starts[-1]), bool((token_pieces != 1).any())
    plan.strips, plan.strip_rows, plan.tiles = len(items[0]), strip_rows, len(items[1])
    parts = [items[0].ravel(), items[1].ravel(), last, starts]
    plan.data = torch.from_numpy(np.concatenate(parts).astype(np.int32)).to(device)
    at = plan.data.data_ptr() + 4 * np.concatenate([[0], np.cumsum([len(part) for part in parts])])
    plan.strips_at, plan.tiles_at, plan.last_at, plan.starts_at = (int(x) for x in at[:4])
    return plan


def attention_shared(q: torch.Tensor, heads: int, cache, block_table: torch.Tensor, plan: SharedPlan, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """The planned step's queries ``q`` [tokens, >= heads * d] (bfloat16, a view of wider rows is fine) over their requests' pages: ``cache`` is a dense
    bfloat16 tensor [pages, 2, kv_heads, page, d] or a :class:`.cache8.Cache8`, ``block_table`` [requests, blocks] int32.  Returns [tokens, heads * d].

    Slots beyond a request's length may hold anything.  What a request's own later tokens hold is masked by weights of 0 for its earlier ones, so
    their values have to be finite."""
    if isinstance(cache, Cache8):
        pages, kv_heads, page_size, head_dim = check_cache8(cache, "attention_shared")
        entries, exponents = cache
    else:
        require_cuda(cache)
        entries, exponents = cache, None
        if cache.dtype != torch.bfloat16 or cache.dim() != 5 or cache.shape[1] != 2 or not cache.is_contiguous():
            raise KernelError("attention_shared: a dense bfloat16 cache [pages, 2, kv_heads, page, d], or a Cache8")
        pages, _, kv_heads, page_size, head_dim = cache.shape
    require_cuda(q, block_table, out)
    if not supported(head_dim, page_size):
        raise KernelError(f"attention_shared: heads of 64 or 128 entries and pages of 8, 16, 32 or 64 positions, not {head_dim} and {page_size}")
    if heads != plan.heads or kv_heads != plan.kv_heads or head_dim != plan.head_dim:
        raise KernelError(f"attention_shared: planned for {plan.heads} heads over {plan.kv_heads} of {plan.head_dim} entries, called with {heads} over {kv_heads} of {head_dim}")
    width = heads * head_dim
    if q.dtype != torch.bfloat16 or q.dim() != 2 or q.shape[0] != plan.tokens or q.shape[1] < width or q.stride(1) != 1:
        raise KernelError(f"attention_shared: bfloat16 queries [{plan.tokens}, {width}] with unit inner stride")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] < plan.rows or not block_table.is_contiguous():
        raise KernelError(f"attention_shared: a dense int32 block table of at least {plan.rows} rows")
    if block_table.shape[1] * page_size < plan.longest:
        raise KernelError(f"attention_shared: a block table of {block_table.shape[1]} pages of {page_size} does not hold {plan.longest} positions")
    if out is None:
        out = torch.empty((plan.tokens, width), dtype=torch.bfloat16, device=q.device)
    elif out.dtype != torch.bfloat16 or out.dim() != 2 or out.shape[0] != plan.tokens or out.shape[1] < width or out.stride(1) != 1:
        raise KernelError(f"attention_shared: the output is a bfloat16 [{plan.tokens}, >= {width}] view")
    if plan.tokens == 0:
        return out
    lib, stream = library("attention_shared", HB_HEAD_DIM=head_dim), stream_ptr()
    pieces = sums = 0
    if plan.joined:
        workspace = torch.empty(max(1, plan.pieces * heads * (head_dim + 2)), dtype=torch.float32, device=q.device)
        pieces = workspace.data_ptr()
        sums = pieces + 4 * plan.pieces * heads * head_dim
    if plan.tiles:
        check(library("attention_shared_tiles", HB_HEAD_DIM=head_dim).hb_attention_shared_tiles(
            ptr(q), q.stride(0), plan.tokens, ptr(out), out.stride(0), ptr(entries), ptr(exponents), ptr(block_table), block_table.shape[1], native.address(plan.tiles_at),
            plan.tiles, native.address(plan.last_at), native.address(plan.starts_at), native.address(pieces), native.address(sums), heads, kv_heads, page_size, pages, f32(scale),
            ptr(status_word(q.device)), stream), "attention_shared")
    if plan.strips:
        check(lib.hb_attention_strips(ptr(q), q.stride(0), ptr(out), out.stride(0), ptr(entries), ptr(exponents), ptr(block_table), block_table.shape[1],
                                      native.address(plan.strips_at), plan.strips, plan.strip_rows, native.address(plan.last_at), native.address(plan.starts_at), native.address(pieces),
                                      native.address(sums), heads, kv_heads, page_size, pages, f32(scale), ptr(status_word(q.device)), stream), "attention_shared")
    if plan.joined:
        check(lib.hb_attention_pieces(native.address(pieces), native.address(sums), native.address(plan.starts_at), ptr(out), out.stride(0), plan.tokens, heads, stream),
              "attention_shared")
    return out
