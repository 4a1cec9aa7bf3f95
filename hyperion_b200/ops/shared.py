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

STRIP_ROWS = 16    # (token, head) rows of a strip
KEY_TILE = 64      # keys of a strip kernel's stage
LEAST_TILES = 3    # of a range that is cut further
BLOCKS_PER_SM = 2  # of the strip kernel


def supported(head_dim: int, page_size: int) -> bool:
    return head_dim in (64, 128) and page_size in (8, 16, 32, 64)


class SharedPlan:
    """What the launches of a step need: the items, the last position each token sees and the first piece of each token, in one int32 tensor."""

    __slots__ = ("tokens", "rows", "heads", "kv_heads", "head_dim", "longest", "pieces", "joined", "strips", "data", "strips_at", "last_at", "starts_at")


def _cut(first, last, tiles_each):
    """Ranges [first, last) cut into shares of about ``tiles_each`` key tiles on tile boundaries: (source range, share's number, first key, last key + 1)."""
    base = first // KEY_TILE
    tiles = -(-last // KEY_TILE) - base
    shares = np.maximum(1, -(-tiles // tiles_each))
    each = -(-tiles // shares)
    shares = -(-tiles // each)  # no share is empty
    source = np.repeat(np.arange(len(first)), shares)
    number = np.arange(len(source)) - np.repeat(np.cumsum(shares) - shares, shares)
    low = np.maximum(first[source], (base[source] + number * each[source]) * KEY_TILE)
    high = np.minimum(last[source], (base[source] + (number + 1) * each[source]) * KEY_TILE)
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
    if length.size and int(length.max()) > 2**31 - 1 - KEY_TILE:
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
    group = heads // kv_heads
    per, across = max(1, STRIP_ROWS // group), kv_heads * -(-group // STRIP_ROWS)  # tokens of a strip, strips beside one another
    cuts = -(-ranges[:, 1] // per)
    tiles = -(-ranges[:, 4] // KEY_TILE) - ranges[:, 3] // KEY_TILE
    work = int((cuts * tiles).sum()) * across
    share = max(LEAST_TILES, -(-work // (BLOCKS_PER_SM * (sms or sm_count(device)))))
    shares, source, number, low, high = _cut(ranges[:, 3], ranges[:, 4], share)
    # a token's pieces: its group's shares, then its own request's
    of_group = np.zeros(requests, dtype=np.int64)
    for k, (*_, first, members) in enumerate(groups):
        of_group[first: first + members] = shares[k]
    of_own = np.zeros(requests, dtype=np.int64)
    of_own[live] = shares[len(groups):]
    number = number + np.concatenate([np.zeros(len(groups), dtype=np.int64), of_group[live]])[source]
    token_pieces = np.repeat(of_group + of_own, n)
    starts = np.concatenate([[0], np.cumsum(token_pieces)])
    # strips: every share of a range for every run of `per` tokens of it
    times = cuts[source]
    at = np.repeat(np.arange(len(source)), times)
    run = np.arange(len(at)) - np.repeat(np.cumsum(times) - times, times)
    tok = ranges[source[at], 0] + run * per
    items = np.stack([tok, np.minimum(per, ranges[source[at], 0] + ranges[source[at], 1] - tok), ranges[source[at], 2], low[at], high[at], number[at]], 1)
    last = np.arange(total) - np.repeat(start[:-1], n) + np.repeat(length - n, n)

    plan = SharedPlan()
    plan.tokens, plan.rows, plan.heads, plan.kv_heads, plan.head_dim = total, requests, heads, kv_heads, head_dim
    plan.longest = int(length[n > 0].max()) if total else 0
    plan.pieces, plan.joined = int(starts[-1]), bool((token_pieces != 1).any())
    plan.strips = len(items)
    flat = np.concatenate([items.ravel(), last, starts]).astype(np.int32)
    plan.data = torch.from_numpy(flat).to(device)
    base = plan.data.data_ptr()
    plan.strips_at, plan.last_at, plan.starts_at = base, base + 4 * items.size, base + 4 * (items.size + total)
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
    if plan.strips:
        check(lib.hb_attention_strips(ptr(q), q.stride(0), ptr(out), out.stride(0), ptr(entries), ptr(exponents), ptr(block_table), block_table.shape[1],
                                      native.address(plan.strips_at), plan.strips, native.address(plan.last_at), native.address(plan.starts_at), native.address(pieces),
                                      native.address(sums), heads, kv_heads, page_size, pages, f32(scale), ptr(status_word(q.device)), stream), "attention_shared")
    if plan.joined:
        check(lib.hb_attention_pieces(native.address(pieces), native.address(sums), native.address(plan.starts_at), ptr(out), out.stride(0), plan.tokens, heads, stream),
              "attention_shared")
    return out
