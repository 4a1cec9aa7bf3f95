"""Rows that stand further apart than 32 bits count: refused, not read elsewhere."""
from __future__ import annotations

import pytest
import torch
from test_shared_attention_gpu import BF, step

from hyperion_b200 import ops
from hyperion_b200.ops.shared import attention_shared, plan_shared

pytestmark = pytest.mark.gpu
MOST = 256 * 64


@pytest.fixture(scope="module")
def apart():
    """Two rows 2^31 entries apart, and 2^32, which 32 bits would count as nothing."""
    memory = torch.zeros(2**32 + MOST, dtype=BF, device="cuda")
    return [memory.as_strided((2, MOST), (stride, 1)) for stride in (2**31, 2**32)]


@pytest.mark.parametrize("counts,lengths,groups", [([1, 1], [40, 40], ()), ([2], [900], ()), ([1, 1], [300, 310], ((0, 2, 256),))])
@pytest.mark.parametrize("heads", [8, 256])  # strips, tiles
def test_attention(apart, heads, counts, lengths, groups):
    q, cache, table = step(counts, lengths, heads, 2, 64, 16, 16, groups)
    plan = plan_shared(counts, lengths, heads, 2, 64, shared=groups)
    assert (plan.tile_blocks > 0) == (heads == 256)
    for rows in apart:
        with pytest.raises(ops.KernelError):
            attention_shared(rows, heads, cache, table, plan, 0.1)
        with pytest.raises(ops.KernelError):
            attention_shared(q, heads, cache, table, plan, 0.1, out=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store(apart, dtype):
    cache = ops.new_cache8(2, 1, 16, 64)
    table, row, position = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.arange(2, dtype=torch.int32, device="cuda")
    for rows in apart if dtype == BF else [apart[1].view(torch.float32)]:
        with pytest.raises(ops.KernelError):
            ops.cache8_store(rows[:, :256], 0, 64, cache, table, row, position)
