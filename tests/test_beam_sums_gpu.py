"""How far the scores of a beam search's selection are from 64 bits.

A row's sum of e^(v - M), M its maximum.  With u = 2^-24: within a look of a thread's, below the maximum A that the thread knows by then, an exponent v L + o is rounded by u of itself, and L, log2(e) as a float, is off by
0.33 u, 0.224 u of itself: together 1.224 u (A - v) of the term.  The hardware's exponential is off by 2^-22 = 4 u, once for the term and once for what the offset o has been rounded by; there are six additions in float
and a product: 7 u.  Everything above that is float64, but each factor e^(m - A) by which what has been added up below a smaller maximum comes below a larger one is the hardware's exponential (4 u) of a difference that is rounded, times L, rounded:
2.224 u (A - m).  The distances of such factors add up to no more than M - v.  A thread's sum takes as many as its maximum rises behind the term, R; then one each from thread to warp, warp to block, piece to lane and lane to row.  So

    |error of the sum| <= (2.224 D + 4 (R + 6) + 7) u   of the sum,    D the mean of M - v with the terms as weights,

as the sum's logarithm is off by, and the scores.  (Terms of second order: 2^-10 of that.)  A score is rounded to float at the end; beams' scores are chosen so that it is near 0."""
from __future__ import annotations

import pytest
import torch

from hyperion_b200.sampling import beam_select

pytestmark = pytest.mark.gpu


def check(logits, rises):
    """One beam a group; ``rises``: how often a thread's maximum may rise behind a term."""
    z = logits.double()
    top, best = z.max(1)
    terms = torch.exp(z - top[:, None])
    total = terms.sum(1)
    distance = (torch.where(terms > 0, terms * (top[:, None] - z), 0.0)).sum(1) / total
    scores = torch.log(total).float()[:, None]  # the best continuation scores nearly 0
    choice = beam_select(logits, scores, 1)
    want = scores[:, 0].double() - torch.log(total)
    assert torch.equal(z.gather(1, choice.tokens.long())[:, 0], top)
    bound = (2.224 * distance + 4 * (rises + 6) + 7) * 2.0 ** -24 * (1 + 2.0 ** -10) + want.abs() * 2.0 ** -24
    error = (choice.scores[:, 0].double() - want).abs()
    assert bool((error <= bound).all()), f"off by up to {(error / bound).max().item():.3f} of what it may be"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [152064, 32001, 5000, 300])
def test_one_outlier_over_a_constant_bulk(vocab, dtype):
    """Errors of what many equal terms share do not average out."""
    rows, random = 64, torch.Generator("cuda").manual_seed(vocab)
    logits = (3 * torch.randn(rows, 1, device="cuda", generator=random)).to(dtype).expand(rows, vocab).contiguous()
    at = torch.randint(0, vocab, (rows, 1), device="cuda", generator=random)
    at[:4, 0] = torch.tensor([0, vocab - 1, vocab // 2, min(vocab - 1, 4096)], device="cuda")
    logits.scatter_(1, at, (logits[:, :1].float() + torch.linspace(0.3, 19.0, rows, device="cuda")[:, None]).to(dtype))
    check(logits, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [152064, 32001, 5000])
@pytest.mark.parametrize("kind", ["normal", "rising", "falling", "far", "masked"])
def test_rows_of_many_kinds(kind, vocab, dtype):
    """Maxima may rise at every look: of 8 warps, each at two runs of 256 or more."""
    rows, random = 16, torch.Generator("cuda").manual_seed(vocab + 1)
    logits = 2.5 * torch.randn(rows, vocab, device="cuda", generator=random)
    if kind in ("rising", "falling"):
        logits = torch.linspace(-20, 0, vocab, device="cuda").expand(rows, vocab) * torch.linspace(0.05, 1, rows, device="cuda")[:, None]
        logits = (logits.flip(1) if kind == "falling" else logits).contiguous()
    elif kind == "far":
        logits += torch.linspace(-3e4, 3e4, rows, device="cuda")[:, None]
    elif kind == "masked":
        logits.masked_fill_(torch.rand(rows, vocab, device="cuda", generator=random) < torch.linspace(0, 0.999, rows, device="cuda")[:, None], float("-inf"))
    check(logits.to(dtype), -(-vocab // (256 * 8 * 2)))
