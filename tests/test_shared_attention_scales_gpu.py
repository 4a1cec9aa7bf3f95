"""A scale that is not above 0 is refused, whatever kernels a step takes."""
from __future__ import annotations

import pytest
from test_shared_attention_gpu import step

from hyperion_b200 import ops
from hyperion_b200.ops.shared import attention_shared, plan_shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan")])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("counts,lengths,groups", [([1], [40], ()), ([1], [900], ()), ([2, 1], [300, 310], ((0, 2, 256),)), ([90], [300], ()), ([0], [40], ())])
def test_scales_that_are_refused(counts, lengths, groups, bits, scale):
    q, cache, table = step(counts, lengths, 8, 2, 64, 16, bits, groups)
    with pytest.raises(ops.KernelError, match="scale"):
        attention_shared(q, 8, cache, table, plan_shared(counts, lengths, 8, 2, 64, shared=groups), scale)
