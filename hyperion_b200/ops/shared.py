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

from .. import host as host_runtime
from .basic import status_word
from .cache8 import Cache8, check_cache8
from .native import KernelError, check, entry, scratch, sm_count, stream_address


TILE_KEYS = 128  # keys of an operand tile


def supported(head_dim: int, page_size: int) -> bool:
    return head_dim in (64, 128) and page_size in (8, 16, 32, 64)


class SharedPlan:
    """What the launches of a step need (csrc/host/shared_plan.hpp): which block of which kernel walks which keys for which tokens, the last position each token sees and its
    pieces, in one int32 tensor."""

    __slots__ = ("requests", "tokens", "heads", "kv_heads", "head_dim", "longest", "pieces", "joined", "strip_blocks", "strip_rows", "tile_blocks", "operand_tiles", "together", "data", "places", "at")


def plan_shared(counts: Sequence[int], lengths: Sequence[int], heads: int, kv_heads: int, head_dim: int, *, shared: Sequence[tuple[int, int, int]] = (),
                device="cuda", sms: int | None = None) -> SharedPlan:
    """Plan a step of ``counts[r]`` queries of request r, whose block table (row r) holds ``lengths[r]`` positions: token i of n sees the first
    ``lengths[r] - n + i + 1`` of them (one with nothing to see comes out as zeros).  ``shared``: (first request, requests, positions) of each group
    of consecutive requests that hold the same pages for their first positions, which all of their queries see; in order, none of them overlapping.
    ``device`` is where the plan is kept, which has to be the device of the step's tensors; ``sms`` its multiprocessors, asked from it when absent.

    The plan is copied there from ordinary memory, so this returns when the current stream has come to the copy: a step is planned before its work is queued."""""
    n, length, groups = (host_runtime.ints(values, np.int64) for values in (counts, lengths, shared))
    if n.ndim != 1 or n.shape != length.shape or (len(groups) and groups.shape[1:] != (3,)):
        raise KernelError("plan_shared: a count of queries and a length for each request, and groups as (first request, requests, positions)")
    lib, sizes = host_runtime.library(), np.empty(18, dtype=np.int64)
    errors = {host_runtime.BAD_ARGUMENT: KernelError}
    host_runtime.check(lib.hb_plan_shared(len(n), host_runtime.address(n), host_runtime.address(length), len(groups), host_runtime.address(groups), heads, kv_heads,
                                          sms or sm_count(device), host_runtime.address(sizes)), errors)
    words = torch.empty(int(sizes[0]), dtype=torch.int32)
    host_runtime.check(lib.hb_plan_shared_take(words.data_ptr(), words.numel()), errors)
    plan = SharedPlan()
    plan.requests, plan.heads, plan.kv_heads, plan.head_dim = len(n), heads, kv_heads, head_dim
    plan.strip_blocks, plan.strip_rows, plan.tile_blocks, plan.tokens, plan.pieces, plan.joined, plan.longest, plan.operand_tiles = sizes[1:9].tolist()
    plan.data = words.to(device)
    plan.together = int(sizes[17])
    plan.places = sizes[9:17].tolist()  # strip items, strip blocks' first items, tile items, tile blocks' first items, last positions, first pieces, first own pieces, operand tiles
    plan.at = [plan.data.data_ptr() + 4 * place for place in plan.places]
    return plan


def attention_shared(q: torch.Tensor, heads: int, cache, block_table: torch.Tensor, plan: SharedPlan, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """The planned step's queries ``q`` [tokens, >= heads * d] (bfloat16, a view of wider rows is fine) over their requests' pages: ``cache`` is a dense
    bfloat16 tensor [pages, 2, kv_heads, page, d] or a :class:`.cache8.Cache8`, ``block_table`` [requests, blocks] int32, ``scale`` above 0.  Rows of ``q``
    stand on 16-byte boundaries, rows of ``out`` on 8-byte ones.  Returns [tokens, heads * d].

    Slots beyond a request's length may hold anything.  What a request's own later tokens hold is masked by weights of 0 for its earlier ones, so
    their values have to be finite.

    A call's scratch memory is 4 * heads * (d + 2) bytes per piece, and over a Cache8 512 * d bytes per 128 positions and key/value head that runs of more than 64 (token, head) rows
    walk (twice those records): up to 16 MB are kept per thread and stream, more is allocated for the call."""""
    if isinstance(cache, Cache8):
        pages, kv_heads, page_size, head_dim = check_cache8(cache, "attention_shared")
        parts, entries, exponents = cache, cache[0].data_ptr(), cache[1].data_ptr()
    else:
        if cache.dtype is not torch.bfloat16 or cache.dim() != 5 or cache.shape[1] != 2 or not cache.is_contiguous():
            raise KernelError("attention_shared: a dense bfloat16 cache [pages, 2, kv_heads, page, d], or a Cache8")
        pages, _, kv_heads, page_size, head_dim = cache.shape
        parts, entries, exponents = (cache,), cache.data_ptr(), 0
    if not supported(head_dim, page_size):
        raise KernelError(f"attention_shared: heads of 64 or 128 entries and pages of 8, 16, 32 or 64 positions, not {head_dim} and {page_size}")
    if heads != plan.heads or kv_heads != plan.kv_heads or head_dim != plan.head_dim:
        raise KernelError(f"attention_shared: planned for {plan.heads} heads over {plan.kv_heads} of {plan.head_dim} entries, called with {heads} over {kv_heads} of {head_dim}")
    tokens, width, shape = plan.tokens, heads * head_dim, q.shape
    if q.dtype is not torch.bfloat16 or len(shape) != 2 or shape[0] != tokens or shape[1] < width or q.stride(1) != 1:
        raise KernelError(f"attention_shared: bfloat16 queries [{tokens}, {width}] with unit inner stride")
    shape = block_table.shape
    if block_table.dtype is not torch.int32 or len(shape) != 2 or shape[0] < plan.requests or not block_table.is_contiguous():
        raise KernelError(f"attention_shared: a dense int32 block table of at least {plan.requests} rows")
    if shape[1] * page_size < plan.longest:
        raise KernelError(f"attention_shared: a block table of {shape[1]} pages of {page_size} does not hold {plan.longest} positions")
    if not scale > 0:
        raise KernelError(f"attention_shared: a scale above 0, not {scale}")
    device = q.device
    if not (q.is_cuda and plan.data.device == block_table.device == parts[0].device == parts[-1].device == device) or (out is not None and out.device != device):
        raise KernelError(f"attention_shared: queries, cache, block table, plan and output on one CUDA device; the plan is on {plan.data.device}, the queries are on {device}")
    if out is None:
        out = torch.empty(tokens, width, dtype=torch.bfloat16, device=device)
    elif out.dtype is not torch.bfloat16 or out.dim() != 2 or out.shape[0] != tokens or out.shape[1] < width or out.stride(1) != 1:
        raise KernelError(f"attention_shared: the output is a bfloat16 [{tokens}, >= {width}] view")
    if tokens == 0:
        return out
    strip_items, strip_first, tile_items, tile_first, last, starts, own, operand_list = plan.at
    out_at, out_stride, stream = out.data_ptr(), out.stride(0), stream_address()
    pieces = sums = operands = 0
    joined = plan.joined and not plan.together
    if joined or plan.operand_tiles:
        for_pieces = (plan.pieces * heads * (head_dim + 2) * 4 + 511) // 512 * 512 if joined else 0
        makes = plan.operand_tiles if exponents else 0  # what runs of many rows walk is made into operands first
        memory, owner = scratch(device, stream, for_pieces + makes * kv_heads * 2 * TILE_KEYS * 2 * head_dim)
        if joined:
            pieces, sums = memory, memory + 4 * plan.pieces * heads * head_dim
        if makes:
            operands = memory + for_pieces
    where = (entries, exponents, block_table.data_ptr(), shape[1])
    what = (last, starts, own, pieces, sums, heads, kv_heads, page_size, pages, scale, status_word(device).data_ptr(), stream)
    if plan.tile_blocks:
        if operands:
            check(entry("attention_shared_tiles", "hb_shared_operands", "pppipipiiipp", head_dim)(
                *where, operand_list, plan.operand_tiles, operands, kv_heads, page_size, pages, status_word(device).data_ptr(), stream), "attention_shared")
        check(entry("attention_shared_tiles", "hb_attention_shared_tiles", "pliplpppippipipppppiiiifpp", head_dim)(
            q.data_ptr(), q.stride(0), tokens, out_at, out_stride, *where, tile_items, tile_first, plan.tile_blocks, operands, plan.operand_tiles, *what), "attention_shared")
    if plan.strip_blocks:
        check(entry("attention_shared", "hb_attention_strips", "plplpppippiiiipppppiiiifppii", head_dim)(
            q.data_ptr(), q.stride(0), out_at, out_stride, *where, strip_items, strip_first, plan.strip_blocks, plan.strip_rows, int(plan.tile_blocks > 0), plan.together, *what, tokens, plan.pieces), "attention_shared")
    elif joined:
        check(entry("attention_shared", "hb_attention_pieces", "ppppliiip", head_dim)(pieces, sums, starts, out_at, out_stride, tokens, plan.pieces, heads, stream), "attention_shared")
    return out
