"""Verification of drafted tokens against the target model's logits, from given random numbers (csrc/verify.cu), and a slow host reference of
the same rule for tests.

A request brings n drafted tokens and n + 1 rows of logits (row i was computed behind draft i - 1).  With p_i = softmax(row_i / temperature) and
the drafter's q_i, draft x_i stands when ``uniform_i * q_i(x_i) < p_i(x_i)``; the first that does not is replaced by a draw from max(p_i - q_i, 0),
and when all stand one more token is drawn from p_n, so that the tokens are distributed as the target's own.  A draw from weights w is
``argmax_v w_v / noise_v`` with exponentially distributed noise.  Temperature 0: a draft stands when it is its row's largest logit, which follows.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from ..ops.basic import status_word
from ..ops.native import KernelError, check, entry, is_bf16, require_cuda, scratch, sm_count, stream_address


CHUNK = 4096  # entries of the vocabulary a block looks through (csrc/verify.cu)


def verify_drafts(logits: torch.Tensor, row_start: torch.Tensor, drafts: torch.Tensor, uniform: torch.Tensor, noise: torch.Tensor, temperature: torch.Tensor, *,
                  most: int, probabilities: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """How many of each request's drafts stand, [requests] int32, and its tokens, [requests, most] int32: the drafts that stand, the token that
    follows them, then -1.

    ``logits`` [rows, vocab] float32 or bfloat16; request r has the rows ``row_start[r]`` to ``row_start[r + 1] - 1`` (int32 [requests + 1]), one more
    than it has drafts; ``most`` is at least the largest such number of rows.  ``drafts`` [rows] int32: the token drafted at each row (a request's
    last one is not read); ``probabilities`` [rows, vocab] float32: the drafter's at that row, or None where it gave none (its token then counts
    with probability 1); ``uniform`` [rows] float32 in [0, 1); ``noise`` [requests, vocab] float32, exponentially distributed, above 0;
    ``temperature`` [requests] float32, 0 for greedy.  At most 65,535 rows and requests.  A draft outside the vocabulary does not stand and is reported (``raise_on_status``)."""
    shape, starts = logits.shape, row_start.shape
    if len(shape) != 2 or len(starts) != 1 or starts[0] < 1:
        raise KernelError("verify_drafts: logits [rows, vocab] and row_start [requests + 1]")
    rows, vocab = shape
    requests = starts[0] - 1
    if logits.stride(1) != 1 or noise.shape != (requests, vocab) or noise.dtype is not torch.float32 or noise.stride(1) != 1:
        raise KernelError("verify_drafts: logits [rows, vocab] and float32 noise [requests, vocab], both with unit inner stride")
    if probabilities is not None and (probabilities.shape != shape or probabilities.dtype is not torch.float32 or probabilities.stride(1) != 1):
        raise KernelError("verify_drafts: the drafter's probabilities are float32 [rows, vocab] with unit inner stride")
    if (row_start.dtype is not torch.int32 or drafts.dtype is not torch.int32 or uniform.dtype is not torch.float32 or temperature.dtype is not torch.float32
            or drafts.shape != (rows,) or uniform.shape != (rows,) or temperature.shape != (requests,)
            or not (row_start.is_contiguous() and drafts.is_contiguous() and uniform.is_contiguous() and temperature.is_contiguous())):
        raise KernelError(f"verify_drafts: dense vectors: row_start int32 [{requests + 1}], drafts int32 [{rows}], uniform float32 [{rows}], temperature float32 [{requests}]")
    if most < 1:
        raise KernelError("verify_drafts: most counts a request's drafts and the token that follows them")
    require_cuda(logits, row_start, drafts, uniform, noise, temperature, probabilities)
    device = logits.device
    accepted, tokens = torch.empty(requests, dtype=torch.int32, device=device), torch.empty(requests, most, dtype=torch.int32, device=device)
    stream = stream_address()
    memory, owner = scratch(device, stream, 8 * (rows * -(-vocab // CHUNK) + 2 * requests))
    check(entry("verify", "hb_verify_drafts", "pilpiiipplpplppppiipp")(
        logits.data_ptr(), is_bf16(logits), logits.stride(0), row_start.data_ptr(), requests, rows, vocab, drafts.data_ptr(),
        probabilities.data_ptr() if probabilities is not None else 0, probabilities.stride(0) if probabilities is not None else 0, uniform.data_ptr(), noise.data_ptr(),
        noise.stride(0), temperature.data_ptr(), memory, accepted.data_ptr(), tokens.data_ptr(), most, sm_count(device), status_word(device).data_ptr(), stream), "verify_drafts")
    return accepted, tokens


def reference_verify(logits: np.ndarray, drafts: Sequence[int], uniform: Sequence[float], noise: np.ndarray, temperature: float,
                     probabilities: Optional[np.ndarray] = None) -> tuple[int, list[int]]:
    """One request by the same rule in float64: (how many drafts stand, those and the token that follows them)."""
    z = np.asarray(logits, dtype=np.float64).copy()
    z[np.isnan(z)] = -np.inf
    z = np.minimum(z, np.finfo(np.float32).max)
    if temperature == 0:
        best = z.argmax(1)
        accepted = next((i for i, x in enumerate(drafts) if x != best[i]), len(drafts))
        return accepted, [int(x) for x in drafts[:accepted]] + [int(best[accepted])]
    top = z.max(1, keepdims=True)
    p = np.where(np.isfinite(top), np.exp((z - np.where(np.isfinite(top), top, 0.0)) / temperature), 0.0)
    p = p / np.maximum(p.sum(1, keepdims=True), np.finfo(np.float64).tiny)
    for i, x in enumerate(drafts):
        q = probabilities[i].astype(np.float64) if probabilities is not None else (np.arange(z.shape[1]) == x).astype(np.float64)
        if not uniform[i] * q[x] < p[i, x]:
            rest = np.maximum(p[i] - q, 0.0)
            return i, [int(y) for y in drafts[:i]] + [int(((rest if rest.max() > 0 else p[i]) / noise).argmax())]
    return len(drafts), [int(x) for x in drafts] + [int((p[len(drafts)] / noise).argmax())]
