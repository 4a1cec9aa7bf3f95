"""How many blocks a step is cut into follows the device's multiprocessors; what comes out does not."""
from __future__ import annotations

import pytest
import torch
from test_cache8_gpu import places
from test_verify_drafts_gpu import case, expected

from hyperion_b200 import ops
from hyperion_b200.ops import cache8
from hyperion_b200.sampling import verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("multiprocessors", [1, 36, 148, 1000])
def test_answers_are_the_same(multiprocessors, monkeypatch):
    c = case([2, 0, 5], 40001, 2)
    asked = []
    monkeypatch.setattr(verify, "sm_count", lambda device: asked.append(device) or multiprocessors)
    accepted, tokens = verify.verify_drafts(**c)
    assert asked
    want = expected(c)
    assert accepted.tolist() == [a for a, _ in want] and tokens.tolist() == [t + [-1] * (c["most"] - len(t)) for _, t in want]
    x = torch.randn(3000, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(torch.bfloat16)
    table, row, position, pages = places(3000, 16, 2)
    first, second = ops.new_cache8(pages, 2, 16, 128), ops.new_cache8(pages, 2, 16, 128)
    ops.cache8_store(x, 0, 256, first, table, row, position)
    back = ops.cache8_load(first, table, row, position)
    monkeypatch.setattr(cache8, "sm_count", lambda device: multiprocessors)
    ops.cache8_store(x, 0, 256, second, table, row, position)
    assert torch.equal(first.codes.view(torch.uint8), second.codes.view(torch.uint8)) and torch.equal(first.exponents, second.exponents)
    assert torch.equal(back, ops.cache8_load(second, table, row, position))
