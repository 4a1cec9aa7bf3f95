"""An infinite temperature: every token that is not masked has the same probability."""
from __future__ import annotations

import pytest
import torch
from test_verify_drafts_gpu import case, expected

from hyperion_b200 import ops
from hyperion_b200.sampling import verify_drafts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_tokens_stay_masked(dtype):
    c = case([2, 0], 6000, 1, dtype, temperatures=(1e30,))  # the rule in 64 bits knows no infinity over infinity: beside 1e30 these logits are equal, too
    c["logits"][:, 50:5900] = -float("inf")
    c["drafts"].clamp_(max=49)
    want = expected(c)
    c["temperature"].fill_(float("inf"))
    accepted, tokens = verify_drafts(**c)
    ops.raise_on_status(tokens.device)
    assert accepted.tolist() == [a for a, _ in want]
    assert tokens.tolist() == [t + [-1] * (3 - len(t)) for _, t in want]
