"""How far attention behind shared positions may be from 64 bits: by the rounding of the result, and little else.

The result is rounded once to bfloat16: 2^-8 of itself (eight significant bits).  Weights carry less: over bfloat16 records, and over 8-bit ones in runs of many rows, they go in two
parts of bfloat16, the first cut off (what it leaves is below 2^-7 of the weight) and the second rounded: 2^-15; over 8-bit records in runs of few rows they are float16: 2^-11.  Float32 adds
the rounding of the scores (some 2^-20 of scores below 8) and of sums of up to 3,000 weights (3,000 * 2^-24 < 2^-12).  Per entry, then: 2^-8 of the result, and of sum_j p_j |v_j| 2^-11,
or 2^-10 where weights are float16.  Weights rounded once to bfloat16 would not pass (``test_the_bound_tells_weights_that_were_rounded_once``): entries whose terms cancel show them."""
from __future__ import annotations

import pytest
import torch
from test_shared_attention_gpu import plain, step

from hyperion_b200 import ops
from hyperion_b200.ops.shared import attention_shared, plan_shared

BF = torch.bfloat16


def beyond(got, want, size, part):
    """Entries that are further from the 64-bit result than they may be."""
    return ((got.double() - want).abs() > 2.0 ** -8 * want.abs() + part * size + 1e-30).sum().item()


STEPS = [([1], [5], ()), ([1, 3], [40, 300], ()), ([2, 1], [3000, 2900], ()), ([1], [9000], ()), ([1, 2, 1], [300, 290, 257], ((0, 3, 250),)),  # strips: whole, in clusters, in pieces, behind a prefix
         ([60], [70], ()), ([90, 40], [90, 1200], ()), ([40] * 2, [1000, 1100], ((0, 2, 900),))]                                               # tiles


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (16, 4, 128)])
@pytest.mark.parametrize("counts,lengths,groups", STEPS)
def test_results_are_off_by_their_rounding(counts, lengths, groups, heads, kv, dim, bits):
    q, cache, table = step(counts, lengths, heads, kv, dim, 16, bits, groups, seed=sum(lengths))
    plan = plan_shared(counts, lengths, heads, kv, dim, shared=groups)
    got = attention_shared(q, heads, cache, table, plan, dim ** -0.5)
    ops.raise_on_status(got.device)
    assert beyond(got, *plain(q, heads, cache, table, counts, lengths, dim ** -0.5), 2.0 ** -10 if bits == 8 and plan.strip_blocks else 2.0 ** -11) == 0


@pytest.mark.parametrize("length", [5, 40, 300])
def test_the_bound_tells_weights_that_were_rounded_once(length):
    """The same rows on the host: with weights in two parts they pass, with weights rounded once to bfloat16 they do not."""
    random = torch.Generator().manual_seed(length)
    q, k, v = (torch.randn(n, 128, generator=random).to(BF).double() for n in (64, length, length))
    p = torch.exp((q @ k.T) * 128 ** -0.5)
    p = p / p.amax(1, keepdim=True)
    want, size = p @ v / p.sum(1, keepdim=True), p @ v.abs() / p.sum(1, keepdim=True)
    first = p.float().view(torch.int32).bitwise_and(-65536).view(torch.float32).double()
    for weights, passes in ((first + (p - first).to(BF).double(), True), (p.to(BF).double(), False)):
        assert (beyond((weights @ v / p.sum(1, keepdim=True)).to(BF), want, size, 2.0 ** -11) == 0) == passes
