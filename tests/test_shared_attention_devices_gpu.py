"""What a step is called with has to be on one device: a plan that was left on the host is refused before anything is launched."""
from __future__ import annotations

import pytest
import torch
from test_shared_attention_gpu import step

from hyperion_b200 import ops
from hyperion_b200.ops.cache8 import Cache8
from hyperion_b200.ops.shared import attention_shared, plan_shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("counts,lengths,groups", [([1], [40], ()), ([1], [900], ()), ([2, 1], [300, 310], ((0, 2, 256),)), ([90], [300], ()), ([0], [40], ())])
def test_a_plan_on_the_host_is_refused(counts, lengths, groups, bits):
    q, cache, table = step(counts, lengths, 8, 2, 64, 16, bits, groups)
    with pytest.raises(ops.KernelError, match="device"):
        attention_shared(q, 8, cache, table, plan_shared(counts, lengths, 8, 2, 64, shared=groups, device="cpu", sms=148), 0.1)


@pytest.mark.parametrize("bits", [8, 16])
def test_tensors_on_the_host_are_refused(bits):
    q, cache, table = step([1], [40], 8, 2, 64, 16, bits)
    good = dict(q=q, heads=8, cache=cache, block_table=table, plan=plan_shared([1], [40], 8, 2, 64), scale=0.1)
    on_host = [dict(q=q.cpu()), dict(block_table=table.cpu()), dict(out=torch.empty(q.shape, dtype=q.dtype)), dict(cache=Cache8(*(part.cpu() for part in cache)) if bits == 8 else cache.cpu())]
    if bits == 8:
        on_host += [dict(cache=cache._replace(codes=cache.codes.cpu())), dict(cache=cache._replace(exponents=cache.exponents.cpu()))]
    for bad in on_host:
        with pytest.raises(ops.KernelError):
            attention_shared(**{**good, **bad})


def test_a_cache_without_pages_is_refused():
    q, _, table = step([1], [40], 8, 2, 64, 16, 8)
    with pytest.raises(ops.KernelError):
        attention_shared(q, 8, ops.new_cache8(0, 2, 16, 64), table, plan_shared([1], [40], 8, 2, 64), 0.1)
