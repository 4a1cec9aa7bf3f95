"""Selection of a beam search's continuations over beams and vocabulary (csrc/beam_select.cu), and a slow host reference of the same rule for tests.

A continuation of beam b by token v scores ``score_b + z_bv - log sum_u e^(z_bu)``, the sum of the log probabilities of its tokens; of equal scores the lowest (beam, token) comes first.
:func:`..ops.beams.beam_reorder` lets the chosen beams go on from what their parents hold."""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from ..ops.native import KernelError, check, entry, is_bf16, scratch, sm_count, stream_address
from ..ops.tally import _check_device, _scratch_size

MOST_BEAMS = 32
MOST_TAKE = 64


class BeamChoice(NamedTuple):
    """Best first, [groups, take] each: the beam that a continuation comes from and its token (int32), and its score (float32)."""
    parents: torch.Tensor
    tokens: torch.Tensor
    scores: torch.Tensor


def beam_select(logits: torch.Tensor, scores: torch.Tensor, take: int) -> BeamChoice:
    """The ``take`` best continuations of each group's beams (as many as it has beams, or twice that where some may end).  ``logits`` [groups * beams, vocab] float32 or bfloat16 with unit inner stride, a
    row per beam; ``scores`` [groups, beams] float32, what the beams have scored so far.  At most 32 beams, ``take`` at most 64, at most 65,535 rows.

    A beam's own tokens come in the order of their logits.  The sums of beams' probabilities are off by some 2^-18 of themselves at most, so continuations of two beams whose scores are closer than 2^-17 may come in either order;
    beams whose logits and scores are the same go by their numbers.

    A logit of -infinity or NaN is no continuation (+infinity counts as the largest number), nor is anything of a beam whose score is -infinity or NaN: a group begins with one beam at 0 and the others at
    -infinity.  Where there are fewer than ``take``, the places left have parent -1, token -1 and score -infinity."""
    held, shape = scores.shape, logits.shape
    if scores.dtype is not torch.float32 or len(held) != 2 or not scores.is_contiguous() or not 1 <= held[1] <= MOST_BEAMS:
        raise KernelError(f"beam_select: scores are dense float32 [groups, beams], 1 to {MOST_BEAMS} beams")
    groups, beams = held
    rows = groups * beams
    if len(shape) != 2 or shape[0] != rows or shape[1] < 1 or logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < shape[1]):
        raise KernelError(f"beam_select: logits [{rows}, vocab] with unit inner stride, rows that do not overlap")
    if not 1 <= take <= MOST_TAKE:
        raise KernelError(f"beam_select: 1 to {MOST_TAKE} continuations, not {take}")
    kind, device, vocab = is_bf16(logits), logits.device, shape[1]
    _check_device("beam_select", logits, scores)
    parents, tokens = torch.empty(groups, take, dtype=torch.int32, device=device), torch.empty(groups, take, dtype=torch.int32, device=device)
    found = scores.new_empty(groups, take)  # (three tensors cost the host 1 us less than views of one)
    if groups == 0:
        return BeamChoice(parents, tokens, found)
    stream, sms = stream_address(), sm_count(device)
    memory, owner = scratch(device, stream, _scratch_size("beam_select", "hb_beam_select_scratch", 0, groups, beams, vocab, take, sms))
    check(entry("beam_select", "hb_beam_select", "pilpiiiipppipp", packed=True)(logits.data_ptr(), kind, logits.stride(0) if rows > 1 else vocab, scores.data_ptr(), groups, beams, vocab, take, parents.data_ptr(), tokens.data_ptr(),
                                                             found.data_ptr(), sms, memory, stream), "beam_select")
    return BeamChoice(parents, tokens, found)


def reference_beam_select(logits: np.ndarray, scores: np.ndarray, take: int) -> list[tuple[int, int, float]]:
    """One group by the same rule in float64: (beam, token, score) of the best continuations, as many as there are."""
    z = np.asarray(logits, dtype=np.float64).copy()
    z[np.isnan(z)] = -np.inf
    z = np.minimum(z, np.finfo(np.float32).max)
    s = np.asarray(scores, dtype=np.float64).copy()
    s[np.isnan(s)] = -np.inf
    s = np.minimum(s, np.finfo(np.float32).max)
    top = z.max(1, keepdims=True)
    alive = np.isfinite(top) & np.isfinite(s)[:, None]
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        total = np.exp(z - np.where(np.isfinite(top), top, 0.0)).sum(1, keepdims=True)
        score = np.where(alive, z + (s[:, None] - (np.where(np.isfinite(top), top, 0.0) + np.log(np.maximum(total, np.finfo(np.float64).tiny)))), -np.inf)
    flat = score.reshape(-1)
    order = np.lexsort((np.arange(flat.size), -flat))[:take]
    return [(int(i) // z.shape[1], int(i) % z.shape[1], float(flat[i])) for i in order if flat[i] > -np.inf]
