"""The largest of a row at temperature 0 where zeros of both signs are the largest: they are equal, and the lowest index is taken."""
from __future__ import annotations

import pytest
import torch
from test_verify_drafts_gpu import case, compare

from hyperion_b200.sampling import verify_drafts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [300, 9000])
def test_zeros_of_both_signs_are_equal(vocab, dtype):
    c = case([2, 1], vocab, 1, dtype, temperatures=(0.0,))
    c["logits"] = -c["logits"].abs() - 1
    c["logits"][:, [17, vocab - 5]] = torch.tensor([-0.0, 0.0], device="cuda", dtype=dtype)
    c["logits"][4, [17, vocab - 5]] = torch.tensor([0.0, -0.0], device="cuda", dtype=dtype)
    c["drafts"].fill_(17)
    compare(c)
    accepted, tokens = verify_drafts(**c)
    assert accepted.tolist() == [2, 1] and tokens.tolist() == [[17, 17, 17], [17, 17, -1]]
