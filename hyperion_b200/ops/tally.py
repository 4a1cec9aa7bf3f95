"""Caches of a fixed budget: attention that keeps its weights (csrc/attention_tallied.cu), the weights of a prompt's queries (csrc/tally_queries.cu), and the eviction of what weighs least
(csrc/evict.cu).

Beside its pages a request has a tally: for each key/value head and slot the weight that its queries have given the slot so far, summed over queries and query heads, and the position of the token
that stands there.  Each key/value head keeps slots of its own; all of a request's heads hold the same number of them, its length.  A prompt's slots hold positions 0, 1, ... as a new tally has them;
keys are stored rotated, so attention does not ask which slot a key stands in, and a slot that eviction fills goes on with its position."""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from .basic import status_word
from .native import KernelError, check, entry, scratch, sm_count, stream_address


LARGEST = 2 ** 31 - 1
LEAST_SCALE, MOST_SCALE = 2.0 ** -100, 2.0 ** 127  # times log2(e) it is a float still


class Tally(NamedTuple):
    """``weights`` float32 and ``positions`` int32, both [requests, kv_heads, capacity], or [layers, requests, kv_heads, capacity]."""
    weights: torch.Tensor
    positions: torch.Tensor


def supported(head_dim: int, page_size: int) -> bool:
    return head_dim in (64, 128) and page_size in (8, 16, 32, 64)


def new_tally(requests: int, kv_heads: int, capacity: int, layers: Optional[int] = None, device="cuda") -> Tally:
    """A tally in which every slot weighs nothing and holds the position of its number, as a prompt's slots do."""
    shape = (requests, kv_heads, capacity) if layers is None else (layers, requests, kv_heads, capacity)
    positions = torch.arange(capacity, dtype=torch.int32, device=device).expand(shape).contiguous()
    return Tally(torch.zeros(shape, device=device), positions)


def _check_tally(tally: Tally, shape: tuple, what: str) -> None:
    """A tally [layers or not, requests, kv_heads, capacity], as it says itself what it holds."""
    weights, positions = tally
    if (weights.shape != shape or positions.shape != shape or weights.dtype is not torch.float32 or positions.dtype is not torch.int32 or not (weights.is_contiguous() and positions.is_contiguous())):
        raise KernelError(f"{what}: a tally is dense float32 weights and int32 positions {[*shape[:-1], 'capacity']}")


def _check_table(what: str, block_table: torch.Tensor, requests: int, page_size: int, longest: Optional[int], capacity: int) -> int:
    """How long a request may be."""
    shape = block_table.shape
    if block_table.dtype is not torch.int32 or len(shape) != 2 or shape[0] < requests or not block_table.is_contiguous():
        raise KernelError(f"{what}: a dense int32 block table of at least {requests} rows")
    holds = shape[1] * page_size
    holds = holds if holds < capacity else capacity
    if longest is None:
        return holds
    if not 0 <= longest <= holds:
        raise KernelError(f"{what}: block table and tally hold {holds} slots, not {longest}")
    return longest


def _check_vector(what: str, name: str, vector: torch.Tensor, size: int) -> None:
    if vector.dtype is not torch.int32 or vector.shape != (size,) or not vector.is_contiguous():
        raise KernelError(f"{what}: {name} is a dense int32 vector of {size}")


def _check_device(what: str, *tensors) -> None:
    """All of them are on the current device."""
    index = tensors[0].get_device()
    if index < 0 or index != torch._C._cuda_getDevice():
        raise KernelError(f"{what}: all tensors on the current CUDA device, not on {tensors[0].device}")
    for tensor in tensors:
        if tensor.get_device() != index:
            raise KernelError(f"{what}: all tensors on the current CUDA device, not on {tensor.device}")


@lru_cache(maxsize=4096)
def _scratch_size(module: str, name: str, head_dim: int, *sizes: int) -> int:
    return entry(module, name, "i" * len(sizes), head_dim, result="l")(*sizes)


def _check_pages(what: str, cache: torch.Tensor, heads: int, q: torch.Tensor, scale: float) -> torch.Size:
    """[pages, 2, kv_heads, page_size, head_dim] of a bfloat16 cache that ``q`` is to look at."""
    shape = cache.shape
    if cache.dtype is not torch.bfloat16 or len(shape) != 5 or shape[1] != 2 or not cache.is_contiguous():
        raise KernelError(f"{what}: a dense bfloat16 cache [pages, 2, kv_heads, page, d]")
    _, _, kv_heads, page_size, head_dim = shape
    if not supported(head_dim, page_size):
        raise KernelError(f"{what}: heads of 64 or 128 entries and pages of 8, 16, 32 or 64 slots, not {head_dim} and {page_size}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise KernelError(f"{what}: {heads} heads over {kv_heads}")
    queries = q.shape
    if q.dtype is not torch.bfloat16 or len(queries) != 2 or queries[1] < heads * head_dim or q.stride(1) != 1:
        raise KernelError(f"{what}: bfloat16 queries [tokens, {heads * head_dim}] with unit inner stride")
    if not LEAST_SCALE <= scale <= MOST_SCALE:
        raise KernelError(f"{what}: a finite scale above 0, not {scale}")
    return shape


def attention_tallied(q: torch.Tensor, heads: int, cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, newest: torch.Tensor, tally: Tally, scale: float, *,
                      longest: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per request: ``q`` [requests, >= heads * d] (bfloat16, a view of wider rows is fine, rows on 16-byte boundaries) over the ``lengths[r]`` (int32) slots of request
    r's pages, the last of which is the new token's own.  ``cache``: dense bfloat16 [pages, 2, kv_heads, page, d]; ``block_table`` [requests, blocks] int32; ``scale`` from 2^-100 to 2^127.  Returns [requests, heads * d], or
    ``out``, a view [requests, >= heads * d] whose rows do not overlap, on 8-byte boundaries.

    What the token gives each slot, summed over the query heads of a key/value head, is added to ``tally`` [requests, kv_heads, capacity]; its own slot enters the tally with what it gives itself and
    with the position ``newest[r]`` (int32).  A request of length 0 comes out as zeros and leaves its tally as it is.  A score of -infinity gives its slot nothing (where all of a head's are, its
    result is zeros); a NaN or +infinity among the scores of a head makes that head's result and its key/value head's weights NaN.

    ``longest``: no request is longer (what table and tally hold, when absent); one that is counts as that long and is reported (``raise_on_status``), unless the bound is 0, where lengths are not looked at.  Work is cut by the
    lengths as they are on the device, so a captured call goes on with other lengths.  Slots beyond a length may hold anything.

    A call's scratch memory is 4 * heads bytes per request and slot up to ``longest``, and 4 * heads * (d + 2) per request and block: up to 16 MB are kept per thread and stream, more is allocated for the call."""
    what = "attention_tallied"
    pages, _, kv_heads, page_size, head_dim = _check_pages(what, cache, heads, q, scale)
    weights, positions = tally
    requests, held, width = q.shape[0], weights.shape, heads * head_dim
    capacity = held[-1] if held else 0
    _check_tally(tally, (requests, kv_heads, capacity), what)
    longest = _check_table(what, block_table, requests, page_size, longest, capacity)
    _check_vector(what, "lengths", lengths, requests)
    _check_vector(what, "newest", newest, requests)
    if out is not None and (out.dtype is not torch.bfloat16 or out.dim() != 2 or out.shape[0] != requests or out.shape[1] < width or out.stride(1) != 1 or (requests > 1 and out.stride(0) < width)):
        raise KernelError(f"{what}: the output is a bfloat16 [{requests}, >= {width}] view with unit inner stride, of rows that do not overlap")
    _check_device(what, q, cache, block_table, lengths, newest, weights, positions, q if out is None else out)
    device = q.device
    if out is None:
        out = q.new_empty(requests, width)
    if requests == 0:
        return out
    if longest == 0:
        out[:, :width].zero_()
        return out
    stream, sms = stream_address(), sm_count(device)
    size = _scratch_size("attention_tallied", "hb_attention_tallied_scratch", head_dim, requests, longest, heads, kv_heads, sms)
    memory, owner = scratch(device, stream, size) if size else (0, None)  # clusters need none
    check(entry("attention_tallied", "hb_attention_tallied", "plplppipiipppiiiiifippp", head_dim, packed=True)(
        q.data_ptr(), q.stride(0) if requests > 1 else width, out.data_ptr(), out.stride(0) if requests > 1 else width, cache.data_ptr(), block_table.data_ptr(), block_table.shape[1], lengths.data_ptr(), requests, longest, weights.data_ptr(),
        positions.data_ptr(), newest.data_ptr(), capacity, heads, kv_heads, page_size, pages, scale, sms, memory, status_word(device).data_ptr(), stream), what)
    return out


def tally_queries(q: torch.Tensor, heads: int, cache: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, tally: Tally, scale: float, *, most: int,
                  longest: Optional[int] = None) -> None:
    """Add to ``tally`` [requests, kv_heads, capacity] what queries give the slots that they see, as :func:`attention_tallied` does for a decoded token, without a result: ``q`` [tokens, >= heads * d] (bfloat16, rows
    on 16-byte boundaries), of which request r has the rows ``starts[r]`` to ``starts[r + 1] - 1`` (int32 [requests + 1]), a whole prompt or the last tokens of one.  They stand in the last of its
    ``lengths[r]`` (int32) slots: query i of n sees the first ``lengths[r] - n + i + 1``, and one with nothing to see gives nothing.  All slots are added to, those of the queries' own tokens too, which have weighed nothing
    before in a new tally; positions are not touched.

    ``most``: no request has more queries; ``longest``: no request is longer (what table and tally hold, when absent).  Queries from ``most`` on, slots from ``longest`` on, and rows that ``q`` does not have are left out
    and reported (``raise_on_status``); the queries that remain see what they would see without the bounds, up to ``longest``.  Where a bound or the number of rows is 0, nothing is looked at.  A score of -infinity gives its slot nothing; a NaN or +infinity among the scores that a
    query sees makes the weights of those slots NaN.

    A call's scratch memory is 16 * heads bytes per query, and 8 * heads more for each of the cuts into which slots go where few queries look at many (two blocks a multiprocessor in all): up to 16 MB are kept
    per thread and stream, more is allocated for the call."""
    what = "tally_queries"
    pages, _, kv_heads, page_size, head_dim = _check_pages(what, cache, heads, q, scale)
    requests, tokens, held = lengths.numel(), q.shape[0], tally.weights.shape
    capacity = held[-1] if held else 0
    _check_tally(tally, (requests, kv_heads, capacity), what)
    longest = _check_table(what, block_table, requests, page_size, longest, capacity)
    _check_vector(what, "lengths", lengths, requests)
    _check_vector(what, "starts", starts, requests + 1)
    if most < 0:
        raise KernelError(f"{what}: most counts a request's queries")
    if heads // kv_heads > 128:
        raise KernelError(f"{what}: at most 128 heads a key/value head, not {heads // kv_heads}")
    _check_device(what, q, cache, block_table, starts, lengths, *tally)
    device = q.device
    most = min(most, tokens)
    if requests == 0 or most == 0 or longest == 0:
        return
    stream, sms = stream_address(), sm_count(device)
    memory, owner = scratch(device, stream, _scratch_size("tally_queries", "hb_tally_queries_scratch", head_dim, tokens, requests, most, longest, heads, kv_heads, sms))
    check(entry("tally_queries", "hb_tally_queries", "plippippiiipiiiiifippp", head_dim, packed=True)(
        q.data_ptr(), q.stride(0) if tokens > 1 else heads * head_dim, tokens, cache.data_ptr(), block_table.data_ptr(), block_table.shape[1], starts.data_ptr(), lengths.data_ptr(), requests, most, longest, tally.weights.data_ptr(), capacity,
        heads, kv_heads, page_size, pages, scale, sms, memory, status_word(device).data_ptr(), stream), what)


def evict(cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, newest: torch.Tensor, tally: Tally, keep: int, *, first: int = 0, recent: int = 0, longest: Optional[int] = None,
          out: Optional[Tally] = None) -> torch.Tensor:
    """Cut requests of more than ``keep`` slots back to ``keep``, the same for every key/value head of every layer, and return the new lengths [requests] int32.  ``cache``: dense
    [layers, pages, 2, kv_heads, page, d] with a ``tally`` [layers, requests, kv_heads, capacity], or both without the layers; any type, records of whole 16 bytes.  ``lengths`` and ``newest`` (the position of each
    request's newest token): int32 [requests].

    Slots whose positions are below ``first`` or among the last ``recent`` rank as an infinite weight, the others by their weights (a NaN as -infinity); of equal ranks the lowest slots stay.  What stays in slots
    from ``keep`` on moves into those below that are left free, in order: keys and values, weights and positions.  Records from the new length on stay as they were; in the tally the slots that were given up
    weigh nothing and have position -1.  The new tally goes to ``out`` where it is given (beside the old one), all of it, with slots behind a request like those given up; else in place, where slots behind a request stay as they were.

    Pages are written in place, so a request's pages may not be another one's as well (up to its length).  ``longest``: no request is longer (what table and tally hold, when absent); one that is counts as that
    long and is reported (``raise_on_status``), unless the bound is 0.  A move from or to a page that is not there is left out and reported.

    A call's scratch memory is 8 bytes for each of the min(keep, longest - keep) moves that a head of a layer and request can have."""
    what, shape = "evict", cache.shape
    layered = len(shape) == 6
    if len(shape) not in (5, 6) or shape[-4] != 2 or not cache.is_contiguous():
        raise KernelError(f"{what}: a dense cache [layers, pages, 2, kv_heads, page, d], or without the layers")
    layers, pages, _, kv_heads, page_size, head_dim = shape if layered else (1, *shape)
    record = head_dim * cache.element_size()
    if page_size & (page_size - 1) or page_size == 0 or record == 0 or record % 16 or record > 65536:
        raise KernelError(f"{what}: pages of a power of two and records of whole 16 bytes, not {page_size} and {record}")
    weights, positions = tally
    to_weights, to_positions = to = tally if out is None else out
    requests, held = lengths.numel(), weights.shape
    capacity = held[-1] if held else 0
    held = (layers, requests, kv_heads, capacity) if layered else (requests, kv_heads, capacity)
    _check_tally(tally, held, what)
    heavy, where, to_heavy, to_where = weights.data_ptr(), positions.data_ptr(), to_weights.data_ptr(), to_positions.data_ptr()
    if to is not tally:
        _check_tally(to, held, what)
        if to_heavy != heavy or to_where != where:  # then beside it
            size = 4 * layers * requests * kv_heads * capacity
            if -size < to_heavy - heavy < size or -size < to_where - where < size:
                raise KernelError(f"{what}: the new tally takes the place of all of the old one, or of none of it")
    longest = _check_table(what, block_table, requests, page_size, longest, capacity)
    _check_vector(what, "lengths", lengths, requests)
    _check_vector(what, "newest", newest, requests)
    if not (1 <= keep <= LARGEST and 0 <= first <= LARGEST and 0 <= recent <= LARGEST):
        raise KernelError(f"{what}: keep from 1, first and recent from 0 to {LARGEST}, not {keep}, {first} and {recent}")
    _check_device(what, cache, block_table, lengths, newest, weights, positions, to_weights, to_positions)
    device = cache.device
    left = torch.empty_like(lengths)
    if requests == 0 or layers == 0 or kv_heads == 0 or longest == 0:
        if to_heavy != heavy:  # nobody has slots
            to_weights.zero_(), to_positions.fill_(-1)
        return left.zero_() if longest == 0 else left.copy_(lengths.clamp(0, min(keep, longest)))
    stream = stream_address()
    memory, owner = scratch(device, stream, _scratch_size("evict", "hb_evict_scratch", 0, layers, requests, kv_heads, longest, keep))
    check(entry("evict", "hb_evict", "piiiiipippiippppiiiipppip", packed=True)(
        cache.data_ptr(), layers, pages, kv_heads, page_size, record, block_table.data_ptr(), block_table.shape[1], lengths.data_ptr(), newest.data_ptr(), requests, longest, heavy,
        where, to_heavy, to_where, capacity, keep, first, recent, left.data_ptr(), memory, status_word(device).data_ptr(), sm_count(device), stream), what)
    return left
