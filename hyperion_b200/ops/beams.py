"""Beams take over what their parents hold (csrc/beam_reorder.cu); :func:`..sampling.beams.beam_select` chooses them."""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from .basic import status_word
from .native import KernelError, check, entry, stream_address
from .tally import _check_device

MOST_TENSORS = 24
MOST_BEAMS = 32


def beam_reorder(parents: torch.Tensor, lengths: torch.Tensor, block_table: Optional[torch.Tensor], caches: Sequence[torch.Tensor], states: Sequence[torch.Tensor] = (), *,
                 state_rows: Optional[torch.Tensor] = None) -> None:
    """Beam j of group g goes on from beam ``parents[g, j]`` (int32 [groups, beams], at most 32 beams; one below 0 leaves its beam as it is): everything in place, any beam the parent of any number.

    Paged caches: ``block_table`` [groups * beams, blocks] int32 has a row per beam, group by group, whose beams all hold ``lengths[g]`` (int32 [groups]) slots.  Entries of full pages become the parent's: pages are
    shared from then on, and whoever hands out pages counts who points to them.  The page behind them, which is not full yet, stays the beam's own (no two beams have the same one there), and the slots of the
    parent's that are filled are copied into it.  ``caches``: dense tensors viewed as [layers, pages, outer, page, inner], all of the same pages and page size (``storage.view(layers, pages, 2 * kv_heads, page, d)``; the codes and
    exponents of an 8-bit cache likewise).

    States: ``states`` are dense [layers, rows, ...], a beam's record copied whole (recurrent states, tallies); a beam's row is its number, or ``state_rows[beam]`` (int32), no two the same.

    At most 24 tensors, each once, none of which overlap.  A parent that is no beam, a row or a page that is not there leaves its beam as it is, and is reported (``raise_on_status``)."""
    what = "beam_reorder"
    if parents.dtype is not torch.int32 or parents.dim() != 2 or not parents.is_contiguous() or parents.shape[1] > MOST_BEAMS:
        raise KernelError(f"{what}: parents are dense int32 [groups, beams], at most {MOST_BEAMS} beams")
    groups, beams = parents.shape
    if lengths.dtype is not torch.int32 or lengths.shape != (groups,) or not lengths.is_contiguous():
        raise KernelError(f"{what}: lengths are a dense int32 vector of {groups}")
    if len(caches) + len(states) > MOST_TENSORS:
        raise KernelError(f"{what}: at most {MOST_TENSORS} tensors, not {len(caches) + len(states)}")
    if caches and block_table is None or block_table is not None and not caches:
        raise KernelError(f"{what}: a block table and the caches that it points into")
    words, spans, rows, page_size, width = [], [], groups * beams, 0, 0
    if block_table is not None:
        width = block_table.shape[-1] if block_table.shape else 0
        if block_table.dtype is not torch.int32 or block_table.shape != (rows, width) or width < 1 or not block_table.is_contiguous():
            raise KernelError(f"{what}: a dense int32 block table of {rows} rows")
        pages, page_size = caches[0].shape[1:4:2] if caches[0].dim() == 5 else (0, 0)
        for cache in caches:
            shape = cache.shape
            if len(shape) != 5 or shape[1] != pages or shape[3] != page_size or pages < 1 or page_size < 1 or not cache.is_contiguous():
                raise KernelError(f"{what}: caches are dense [layers, pages, outer, page, inner], all of the same pages and page size")
            at, layers, _, outer, _, inner = cache.data_ptr(), *shape
            slot = inner * cache.element_size()
            words += (at, layers, pages, outer, page_size, slot, 0)
            spans.append((at, at + layers * pages * outer * page_size * slot))
    if state_rows is not None and (state_rows.dtype is not torch.int32 or state_rows.shape != (rows,) or not state_rows.is_contiguous()):
        raise KernelError(f"{what}: state_rows is a dense int32 vector of {rows}")
    for state in states:
        if state.dim() < 2 or state.shape[1] != states[0].shape[1] or not state.is_contiguous() or (state.shape[1] != rows if state_rows is None else state.shape[1] < 1):
            raise KernelError(f"{what}: states are dense [layers, {rows if state_rows is None else 'rows'}, ...]")
        layers, places = state.shape[:2]
        at, size = state.data_ptr(), state.numel() * state.element_size()
        words += (at, layers, places, 1, 1, size // max(1, layers * places), 1)
        spans.append((at, at + size))
    if len(spans) > 1:
        spans.sort()
        end = 0
        for start, its_end in spans:
            if start < end and start < its_end:
                raise KernelError(f"{what}: a tensor once only, and no two that overlap")
            end = max(end, its_end)
    tensors = [parents, lengths, *caches, *states]
    if block_table is not None:
        tensors.append(block_table)
    if state_rows is not None:
        tensors.append(state_rows)
    _check_device(what, *tensors)
    if rows == 0 or not words:
        return
    described = (ctypes.c_longlong * len(words))(*words)
    check(entry("beam_reorder", "hb_beam_reorder", "ppiipiipippp", packed=True)(
        parents.data_ptr(), lengths.data_ptr(), groups, beams, block_table.data_ptr() if block_table is not None else 0, width, page_size,
        ctypes.addressof(described), len(words) // 7, state_rows.data_ptr() if state_rows is not None else 0,
        status_word(parents.device).data_ptr(), stream_address()), what)
