"""A key that takes nearly all of a row's weight and brings little or nothing to an entry, before thousands of keys whose weights are small beside its own: the entry is theirs.

Tolerance: the result's rounding (up to 2^-8 of it, and results are well below sum_j p_j |v_j| here: 3,000 terms of either sign), and the weights'.  Over 8-bit records, runs of many rows carry
weights in two parts of bfloat16 (2^-15 of each); runs of few rows carry them in float16, 2^8 above one for the largest: 2^-11 of a weight, and 2^-25 where it lies below 2^-14.  With
the largest weight 2^29 times the others that is up to 2^-4 of one weight, and of the sum of 3,000 of random size 2^-4 / sqrt(3 * 3,000) < 2^-10.  2^-8 of sum_j p_j |v_j| holds both, and
what float32 adds."""
from __future__ import annotations

import pytest
import torch
from test_shared_attention_gpu import BF, plain

from hyperion_b200 import ops
from hyperion_b200.ops.cache8 import Cache8
from hyperion_b200.ops.shared import attention_shared, plan_shared

pytestmark = pytest.mark.gpu
PAGE = 16


def sink(length, heads, kv, dim, rows, weight, values, seed=0):
    """One request whose first key has a score of ``weight`` * ln 2 beside scores around zero, and a value that is zero in all entries but one (``values`` "zero"), or 2^-11 of the others'
    size (``values`` "tiny")."""
    random = torch.Generator("cuda").manual_seed(seed)
    pages = -(-length // PAGE)
    x = torch.randn(pages, 2, kv, PAGE, dim, device="cuda", generator=random)
    x[:, 0] *= 2.0 ** -4
    cache = Cache8((x * 64).clamp(-448, 448).to(torch.float8_e4m3fn), torch.full((pages, 2, kv, PAGE), -6, dtype=torch.int8, device="cuda"))
    codes = cache.codes.view(torch.uint8)
    codes[0, 0, :, 0] = 0
    codes[0, 0, :, 0, 0] = torch.tensor([weight * 0.6931], device="cuda").mul(8).to(torch.float8_e4m3fn).view(torch.uint8)
    cache.exponents[0, 0, :, 0] = -3
    if values == "zero":
        codes[0, 1, :, 0] = 0
        codes[0, 1, :, 0, 5] = 0x7E
    else:
        cache.exponents[0, 1, :, 0] -= 11
    q = torch.randn(rows, heads, dim, device="cuda", generator=random) * 0.1
    q[:, :, 0] = 1.0
    return q.view(rows, -1).to(BF), cache, torch.arange(pages, dtype=torch.int32, device="cuda").view(1, pages)


@pytest.mark.parametrize("values", ["zero", "tiny"])
@pytest.mark.parametrize("weight", [20, 24, 28])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (16, 4, 128)])
@pytest.mark.parametrize("rows", [1, 40])
def test_small_weights_beside_a_large_one(rows, heads, kv, dim, weight, values):
    length = 3000 + rows
    q, cache, table = sink(length, heads, kv, dim, rows, weight, values)
    plan = plan_shared([rows], [length], heads, kv, dim)
    assert (plan.tile_blocks > 0) == (rows > 1)
    check(q, heads, cache, table, plan, [rows], [length])


@pytest.mark.parametrize("values", ["zero", "tiny"])
@pytest.mark.parametrize("weight", [33, 40, 60])
def test_much_smaller_weights_in_runs_of_many_rows(weight, values):
    q, cache, table = sink(3040, 16, 4, 128, 40, weight, values, seed=1)
    check(q, 16, cache, table, plan_shared([40], [3040], 16, 4, 128), [40], [3040])


def check(q, heads, cache, table, plan, counts, lengths):
    got = attention_shared(q, heads, cache, table, plan, 1.0)
    ops.raise_on_status(got.device)
    want, size = plain(q, heads, cache, table, counts, lengths, 1.0)
    assert ((got.double() - want).abs() <= 2.0 ** -8 * size).all(), float(((got.double() - want).abs() / size).max())
