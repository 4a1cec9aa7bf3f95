"""Eviction where a bound leaves nothing of any request: a new tally in a place of its own is written all the same."""
from __future__ import annotations

import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops import Tally, evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [0, 3])
def test_a_bound_of_zero_slots(layers):
    shape = (layers, 2, 4, 40) if layers else (2, 4, 40)
    cache = torch.randn(*([layers] if layers else []), 9, 2, 4, 16, 32, device="cuda")
    given = cache.clone()
    table, lengths = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    old = Tally(torch.rand(shape, device="cuda"), torch.randint(0, 99, shape, dtype=torch.int32, device="cuda"))
    kept = Tally(*(x.clone() for x in old))
    new = Tally(torch.full(shape, 3.0, device="cuda"), torch.full(shape, 3, dtype=torch.int32, device="cuda"))
    for longest in (0, 40):
        new.weights.fill_(3.0), new.positions.fill_(3)
        assert evict(cache, table, lengths, lengths, old, 5, longest=longest, out=new).tolist() == [0, 0]
        assert bool((new.weights == 0).all()) and bool((new.positions == -1).all())
        assert evict(cache, table, lengths, lengths, old, 5, longest=longest).tolist() == [0, 0]
        assert torch.equal(old.weights, kept.weights) and torch.equal(old.positions, kept.positions) and torch.equal(cache, given)
    ops.raise_on_status(cache.device)
